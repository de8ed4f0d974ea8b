// yl_layernorm.cu -- LayerNorm over the last axis of [rows][cols] fp32,
// forward and backward.
//
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  r = 1 / sqrt(var + eps),
//   h = (x - mean) r,  y = h gamma + beta;
//   t = dy gamma,  dx = r (t - mean(t) - h mean(t h)) (+ addend),
//   dgamma = sum over rows of dy h,  dbeta = sum over rows of dy.
#include <algorithm>

#include "yl_internal.h"
#include "yl_muon.h"
#include "yume_c.h"

using namespace yl;

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block, the same value in every thread.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

// mean (as a pair: the rounded mean and what it is short of) and 1 / sqrt(var + eps)
__device__ __forceinline__ void row_stats(const float* x, int cols, float eps, float* red,
                                          float* mean, float* short_of, float* rstd) {
  float s = 0.f;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) s += x[c];
  const float m = block_sum(s, red) / cols;
  float d1 = 0.f, d2 = 0.f;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const float d = x[c] - m;
    d1 += d;
    d2 += d * d;
  }
  const float e = block_sum(d1, red) / cols;
  const float var = fmaxf(block_sum(d2, red) / cols - e * e, 0.f);
  *mean = m;
  *short_of = e;
  *rstd = 1.f / sqrtf(var + eps);
}

__global__ void __launch_bounds__(kThreads)
    ln_fwd_kernel(const float* __restrict__ x, long long ldx, long long rows, int cols, float eps,
                  const float* __restrict__ gamma, const float* __restrict__ beta,
                  float* __restrict__ y, long long ldy, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out) {
  __shared__ float red[32];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* xr = x + r * ldx;
    float m, e, rs;
    row_stats(xr, cols, eps, red, &m, &e, &rs);
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float h = ((xr[c] - m) - e) * rs;
      y[r * ldy + c] = h * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f);
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = m + e;
      if (rstd_out) rstd_out[r] = rs;
    }
  }
}

// dx of each row, and the row's statistics for the column sums.
__global__ void __launch_bounds__(kThreads)
    ln_bwd_dx_kernel(const float* __restrict__ x, long long ldx, const float* __restrict__ dy,
                     long long lddy, long long rows, int cols, float eps,
                     const float* __restrict__ gamma, const float* __restrict__ mean,
                     const float* __restrict__ rstd, const float* addend, long long ldadd,
                     float* dx, long long lddx, float2* __restrict__ stats) {
  __shared__ float red[32];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* xr = x + r * ldx;
    const float* dr = dy + r * lddy;
    float m, e = 0.f, rs;
    if (mean) {
      m = mean[r];
      rs = rstd[r];
    } else {
      row_stats(xr, cols, eps, red, &m, &e, &rs);
      m += e;
    }
    if (threadIdx.x == 0) stats[r] = make_float2(m, rs);
    if (!dx) continue;
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float t = dr[c] * (gamma ? gamma[c] : 1.f);
      s1 += t;
      s2 += t * (xr[c] - m) * rs;
    }
    const float c1 = block_sum(s1, red) / cols, c2 = block_sum(s2, red) / cols;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float t = dr[c] * (gamma ? gamma[c] : 1.f);
      const float h = (xr[c] - m) * rs;
      float v = rs * (t - c1 - h * c2);
      if (addend) v += addend[r * ldadd + c];
      dx[r * lddx + c] = v;
    }
  }
}

// part[chunk][2][cols]: sums over the rows of one chunk
__global__ void ln_bwd_cols_kernel(const float* __restrict__ x, long long ldx,
                                   const float* __restrict__ dy, long long lddy, long long rows,
                                   int cols, const float2* __restrict__ stats,
                                   double* __restrict__ part) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  double g = 0.0, b = 0.0;
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    const float2 st = stats[r];
    const float d = dy[r * lddy + c];
    g += (double)(d * ((x[r * ldx + c] - st.x) * st.y));
    b += (double)d;
  }
  part[(2LL * blockIdx.y) * cols + c] = g;
  part[(2LL * blockIdx.y + 1) * cols + c] = b;
}

__global__ void ln_bwd_cols_final_kernel(const double* __restrict__ part, int chunks, int cols,
                                         float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  double g = 0.0, b = 0.0;
  for (int k = 0; k < chunks; ++k) {
    g += part[(2LL * k) * cols + c];
    b += part[(2LL * k + 1) * cols + c];
  }
  if (dgamma) dgamma[c] = (float)g;
  if (dbeta) dbeta[c] = (float)b;
}

bool aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }

yl_status check_ln(yl_ctx* ctx, const char* who, long long rows, int cols, float eps) {
  YL_CHECK(ctx, YL_ERR_INVALID, "%s: ctx is NULL", who);
  YL_CHECK(rows >= 0 && cols >= 1, YL_ERR_SHAPE, "%s: %lld rows of %d columns", who, rows, cols);
  YL_CHECK(eps >= 0.f, YL_ERR_INVALID, "%s: eps %g is negative or NaN", who, (double)eps);
  return YL_OK;
}

}  // namespace

extern "C" {

yl_status yl_layernorm_fwd(yl_ctx* ctx, const float* x, long long ldx, long long rows, int cols,
                           float eps, const float* gamma, const float* beta, float* y,
                           long long ldy, float* mean_out, float* rstd_out) {
  YL_TRY(check_ln(ctx, "yl_layernorm_fwd", rows, cols, eps));
  if (rows == 0) return YL_OK;
  YL_CHECK(x && y, YL_ERR_INVALID, "yl_layernorm_fwd: NULL argument");
  YL_CHECK(aligned4(x) && aligned4(gamma) && aligned4(beta) && aligned4(y) && aligned4(mean_out) &&
               aligned4(rstd_out),
           YL_ERR_INVALID, "yl_layernorm_fwd: a pointer is not a multiple of 4 bytes");
  YL_CHECK(ldx >= cols && ldy >= cols, YL_ERR_SHAPE,
           "yl_layernorm_fwd: row strides %lld, %lld are smaller than %d columns", ldx, ldy, cols);
  YL_CHECK((x == y && ldx == ldy) || !rows_overlap(x, ldx, rows, cols, y, ldy, rows, cols),
           YL_ERR_INVALID, "yl_layernorm_fwd: y overlaps x");
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  const unsigned grid = (unsigned)std::min<long long>(rows, ctx->num_sms * 16LL);
  ln_fwd_kernel<<<grid, kThreads, 0, ctx->stream>>>(x, ldx, rows, cols, eps, gamma, beta, y, ldy,
                                                    mean_out, rstd_out);
  return check_launch("ln_fwd_kernel");
}

yl_status yl_layernorm_bwd(yl_ctx* ctx, const float* x, long long ldx, const float* dy,
                           long long lddy, long long rows, int cols, float eps, const float* gamma,
                           const float* mean, const float* rstd, const float* addend,
                           long long ldadd, float* dx, long long lddx, float* dgamma,
                           float* dbeta) {
  YL_TRY(check_ln(ctx, "yl_layernorm_bwd", rows, cols, eps));
  YL_CHECK((mean == nullptr) == (rstd == nullptr), YL_ERR_INVALID,
           "yl_layernorm_bwd: mean and rstd are given together or not at all");
  if (rows == 0) {
    DeviceGuard dev(ctx->device);
    YL_CUDA(dev.status());
    if (dgamma) YL_CUDA(cudaMemsetAsync(dgamma, 0, cols * sizeof(float), ctx->stream));
    if (dbeta) YL_CUDA(cudaMemsetAsync(dbeta, 0, cols * sizeof(float), ctx->stream));
    return YL_OK;
  }
  YL_CHECK(x && dy, YL_ERR_INVALID, "yl_layernorm_bwd: NULL argument");
  YL_CHECK(aligned4(x) && aligned4(dy) && aligned4(gamma) && aligned4(mean) && aligned4(rstd) &&
               aligned4(addend) && aligned4(dx) && aligned4(dgamma) && aligned4(dbeta),
           YL_ERR_INVALID, "yl_layernorm_bwd: a pointer is not a multiple of 4 bytes");
  YL_CHECK(ldx >= cols && lddy >= cols && (!addend || ldadd >= cols) && (!dx || lddx >= cols),
           YL_ERR_SHAPE, "yl_layernorm_bwd: a row stride is smaller than %d columns", cols);
  YL_CHECK(!rows_overlap(x, ldx, rows, cols, dx, lddx, rows, cols) &&
               !rows_overlap(dy, lddy, rows, cols, dx, lddx, rows, cols) &&
               ((addend == dx && ldadd == lddx) ||
                !rows_overlap(addend, ldadd, rows, cols, dx, lddx, rows, cols)),
           YL_ERR_INVALID, "yl_layernorm_bwd: dx overlaps an input");
  if (!dx && !dgamma && !dbeta) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  const int chunks = (int)std::min<long long>(rows, 256);
  ScratchCarver carve;
  const size_t o_st = carve.take(rows * sizeof(float2));
  const size_t o_part = carve.take((size_t)chunks * 2 * cols * sizeof(double));
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, carve.offset, &ws));
  const unsigned grid = (unsigned)std::min<long long>(rows, ctx->num_sms * 16LL);
  ln_bwd_dx_kernel<<<grid, kThreads, 0, ctx->stream>>>(x, ldx, dy, lddy, rows, cols, eps, gamma,
                                                       mean, rstd, addend, ldadd, dx, lddx,
                                                       (float2*)(ws + o_st));
  YL_TRY(check_launch("ln_bwd_dx_kernel"));
  if (dgamma || dbeta) {
    const dim3 g2((cols + 127) / 128, chunks);
    ln_bwd_cols_kernel<<<g2, 128, 0, ctx->stream>>>(x, ldx, dy, lddy, rows, cols,
                                                    (const float2*)(ws + o_st),
                                                    (double*)(ws + o_part));
    YL_TRY(check_launch("ln_bwd_cols_kernel"));
    ln_bwd_cols_final_kernel<<<(cols + 127) / 128, 128, 0, ctx->stream>>>(
        (const double*)(ws + o_part), chunks, cols, dgamma, dbeta);
    YL_TRY(check_launch("ln_bwd_cols_final_kernel"));
  }
  return work.done();
}

}  // extern "C"
