// Kernels of the selective scan for bf16.
#include "selective_scan_kernels.h"

int fc_scan_ends_bf16(fc_context *ctx, const fc_scan_run &r) { return scan_ends<FC_BF16>(ctx, r); }
int fc_scan_answers_bf16(fc_context *ctx, const fc_scan_run &r) { return scan_answers<FC_BF16>(ctx, r); }
int fc_scan_step_bf16(fc_context *ctx, const fc_scan_run &r) { return scan_step<FC_BF16>(ctx, r); }
int fc_scan_gradients_bf16(fc_context *ctx, const fc_scan_run &r) { return scan_gradients<FC_BF16>(ctx, r); }
