// yl_muon.h -- internal API of the Newton-Schulz / Muon kernels.
#pragma once
#include "yl_internal.h"

namespace yl {

// Longest side of a matrix.
constexpr int kNsMaxSide = 65536;

struct MuonStep {
  float lr = 0.02f, momentum = 0.95f;
  int nesterov = 1;
  float weight_decay = 0.f;
  int steps = 5;
  float eps = 1e-7f, grad_scale = 1.f, clip_max_norm = 0.f;
  int sanitize = 0;
};

// coeffs: three per step, or null for the quintic (3.4445, -4.7750, 2.0315).
// Whether the operators take these steps.
yl_status check_steps(const char* who, int steps, const float* coeffs);
yl_status newton_schulz(yl_ctx* ctx, const yl_ns_matrix* table, int count, int steps,
                        const float* coeffs, float eps);
// norm: device scalar with the gradients' global norm for the clip, or null to
// measure it over this table; norm_out (device, optional) receives that.
yl_status muon_multi(yl_ctx* ctx, const yl_muon_tensor* table, int count, const MuonStep& st,
                     const float* coeffs, const float* norm, float* norm_out);

// L2 norm of n scaled (and sanitized) gradients -> norm_out (device).
yl_status grad_norm(yl_ctx* ctx, const float* g, long long n, float grad_scale, int sanitize,
                    float* norm_out);

// Whether two strided row blocks of floats share an element (true as well when
// their row strides differ and their extents overlap).
bool rows_overlap(const float* a, long long lda, long long rows_a, long long cols_a,
                  const float* b, long long ldb, long long rows_b, long long cols_b);

}  // namespace yl
