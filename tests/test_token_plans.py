"""Shapes and plans of the operators on tokens: what they refuse, and their layout.  No GPU needed."""
import ctypes as C
import os
import subprocess

import pytest

from fastconv_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"fc_group_norm_shape": capi.GroupNormShape, "fc_group_norm_plan": capi.GroupNormPlan, "fc_rotary_shape": capi.RotaryShape,
               "fc_linear_attention_shape": capi.LinearAttentionShape, "fc_linear_attention_plan": capi.LinearAttentionPlan}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fastconv_hip.h"', 'int main(void) {']
    for cname, ct in structs.items():
        lines.append('printf("%s sizeof %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in ct._fields_]
    lines.append('printf("values F32 %d\\nvalues BF16 %d\\nvalues F16 %d\\nvalues ACT_NONE %d\\nvalues ACT_RELU %d\\nvalues ACT_SILU %d\\n'
                 'values ACT_GELU %d\\nvalues ROTARY_AXES %d\\n", FC_F32, FC_BF16, FC_F16, FC_ACT_NONE, FC_ACT_RELU, FC_ACT_SILU, '
                 'FC_ACT_GELU, FC_ROTARY_AXES); return 0;}')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    seen = 0
    for line in subprocess.check_output([str(exe)], text=True).splitlines():
        cname, field, value = line.split()
        if cname == "values":
            assert getattr(capi, field) == int(value), field
        elif field == "sizeof":
            assert C.sizeof(structs[cname]) == int(value), cname
        else:
            assert getattr(structs[cname], field).offset == int(value), (cname, field)
        seen += 1
    assert seen == sum(len(ct._fields_) + 1 for ct in structs.values()) + 8


def plan_of(make, plan, shape, **change):
    for name, v in change.items():
        setattr(shape, name, v)
    return make(C.byref(shape), C.byref(plan))


def norm(**change):
    plan = capi.GroupNormPlan()
    return plan_of(capi.load_cdll().fc_group_norm_make_plan, plan, capi.GroupNormShape.packed(2, 100, 64, 8, capi.BF16, capi.ACT_SILU), **change), plan


def attention(**change):
    plan = capi.LinearAttentionPlan()
    return plan_of(capi.load_cdll().fc_linear_attention_make_plan, plan, capi.LinearAttentionShape.packed(2, 100, 8, 4, 64, 64, capi.BF16, 0.125),
                   **change), plan


@pytest.mark.parametrize("field,value,status", [
    ("N", 0, -1), ("P", 0, -1), ("C", 0, -1), ("G", 0, -1), ("G", 7, -1), ("dtype", 3, -1), ("dtype", -1, -1), ("act", 4, -1),
    ("eps", -1e-5, -1), ("eps", float("nan"), -1), ("x_image", -1, -1), ("x_pixel", -1, -1), ("y_image", -1, -1), ("y_pixel", -1, -1),
    ("P", 1 << 60, -6)])
def test_group_norm_refuses(field, value, status):
    assert norm(**{field: value})[0] == status


def test_group_norm_limit_is_the_channels_of_a_group():
    assert norm(C=4096, G=1)[0] == 0
    assert norm(C=4097, G=1)[0] == -6
    assert norm(C=4097 * 4, G=4097)[0] == 0


@pytest.mark.parametrize("field,value,status", [
    ("B", 0, -1), ("T", 0, -1), ("H", 0, -1), ("Hkv", 0, -1), ("Hkv", 3, -1), ("Dk", 0, -1), ("Dv", 0, -1), ("dtype", 3, -1),
    ("scale", float("inf"), -1), ("scale", float("nan"), -1), ("q_token", -1, -1), ("o_head", -1, -1), ("Dk", 257, -6), ("Dv", 257, -6),
    ("T", 1 << 40, -6), ("B", 1 << 30, -6)])
def test_linear_attention_refuses(field, value, status):
    assert attention(**{field: value})[0] == status


def test_null_arguments_are_refused():
    lib = capi.load_cdll()
    assert lib.fc_group_norm_make_plan(None, C.byref(capi.GroupNormPlan())) == -1
    assert lib.fc_linear_attention_make_plan(None, C.byref(capi.LinearAttentionPlan())) == -1
    s = capi.GroupNormShape.packed(1, 1, 1, 1)
    assert lib.fc_group_norm_make_plan(C.byref(s), None) == -1
    # a call without a context
    assert lib.fc_group_norm(None, None, None, None, None, None, None, None, None) == -5
    assert lib.fc_rotary(None, None, None, None, None, None, 0, None, None) == -5
    assert lib.fc_linear_attention(None, None, *([None] * 9)) == -5


def test_spans_are_whole_groups_that_fit():
    for c, g in ((64, 32), (192, 32), (63, 7), (4100, 2), (4097 * 2, 4097), (6153, 3), (1 << 16, 16), (5, 5)):
        for dtype in (capi.F32, capi.BF16):
            rc, plan = norm(C=c, G=g, x_pixel=c, y_pixel=c, dtype=dtype)
            assert rc == 0 and 0 < plan.span <= 4096 and plan.span % (c // g) == 0 and plan.chunks >= 1


def test_launches_stay_below_their_limit():
    assert norm(N=1 << 24)[0] == -6
    rc, plan = norm(N=(1 << 21) - 1)
    assert rc == 0 and plan.resident == 32
    rc, plan = norm(N=1 << 21)      # two resident workgroups of 1024 threads an image would be 2^32 threads
    assert rc == 0 and plan.resident == 0
    assert attention(B=(1 << 18) - 1, T=1)[0] == 0
    assert attention(B=1 << 18, T=1)[0] == -6


def test_every_norm_has_a_plan_of_whole_groups():
    for n in (1, 7, 300):
        for p in (1, 49, 1225, 12544, 60000):
            for c, g in ((1, 1), (7, 7), (32, 32), (48, 6), (96, 32), (130, 13), (256, 1), (512, 32), (4096, 1), (5000, 1250)):
                for dtype in (capi.F32, capi.BF16):
                    rc, plan = norm(N=n, P=p, C=c, G=g, dtype=dtype, x_image=p * c, x_pixel=c, y_image=p * c, y_pixel=c)
                    assert rc == 0 and plan.span % (c // g) == 0 and plan.chunks >= 1
                    for span in (plan.resident, plan.resident_backward):
                        assert span == 0 or (c % span == 0 and span % (c // g) == 0 and span % (4 if dtype == capi.F32 else 8) == 0)


def test_sequences_are_cut_for_the_wavefronts_that_are_launched():
    """About 2048 wavefronts fill the chip.  A head of 64 takes two in 16 bits; four in fp32, and in half where four channels lie in no access."""
    def packed(B, T, H, Dk, Dv, dtype, **change):
        plan = capi.LinearAttentionPlan()
        shape = capi.LinearAttentionShape.packed(B, T, H, H, Dk, Dv, dtype)
        assert plan_of(capi.load_cdll().fc_linear_attention_make_plan, plan, shape, **change) == 0
        return plan.segments
    for dtype, wavefronts in ((capi.BF16, 2), (capi.F16, 2), (capi.F32, 4)):
        for B, T, H in ((8, 2048, 32), (1, 11760, 8), (8, 1225, 8), (4, 3136, 16)):
            segments = packed(B, T, H, 64, 64, dtype)
            assert B * H * segments * wavefronts <= 2048 and (segments == 1 or B * H * (segments + 1) * wavefronts > 1024), (dtype, B, T, H, segments)
    assert packed(8, 2048, 32, 64, 64, capi.F32) == 1                 # three parts or none
    assert packed(1, 11760, 8, 32, 32, capi.F32) == packed(1, 11760, 8, 64, 64, capi.BF16) > packed(1, 11760, 8, 64, 64, capi.F32)
    assert packed(4, 3136, 16, 63, 61, capi.F16) == packed(4, 3136, 16, 64, 64, capi.F32)
    assert packed(4, 3136, 16, 64, 64, capi.F16, q_token=16 * 64 + 1) == packed(4, 3136, 16, 64, 64, capi.F32)
