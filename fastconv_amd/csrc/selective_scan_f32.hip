// Kernels of the selective scan for fp32.
#include "selective_scan_kernels.h"

int fc_scan_ends_f32(fc_context *ctx, const fc_scan_run &r) { return scan_ends<FC_F32>(ctx, r); }
int fc_scan_answers_f32(fc_context *ctx, const fc_scan_run &r) { return scan_answers<FC_F32>(ctx, r); }
int fc_scan_step_f32(fc_context *ctx, const fc_scan_run &r) { return scan_step<FC_F32>(ctx, r); }
int fc_scan_gradients_f32(fc_context *ctx, const fc_scan_run &r) { return scan_gradients<FC_F32>(ctx, r); }
