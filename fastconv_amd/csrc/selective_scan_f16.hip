// Kernels of the selective scan for half.
#include "selective_scan_kernels.h"

int fc_scan_ends_f16(fc_context *ctx, const fc_scan_run &r) { return scan_ends<FC_F16>(ctx, r); }
int fc_scan_answers_f16(fc_context *ctx, const fc_scan_run &r) { return scan_answers<FC_F16>(ctx, r); }
int fc_scan_step_f16(fc_context *ctx, const fc_scan_run &r) { return scan_step<FC_F16>(ctx, r); }
int fc_scan_gradients_f16(fc_context *ctx, const fc_scan_run &r) { return scan_gradients<FC_F16>(ctx, r); }
