// yl_muon.cu -- Newton-Schulz orthogonalisation of a table of matrices and the
// Muon step built on it.
//
//   X0 = U / (|U|_F + eps);  A = X X^T,  X <- (a I + b A + c A^2) X, `steps`
//   times, with X taken so that its rows are its shorter side.  Every singular
//   value s of X0 goes to p(p(...p(s))), p(s) = a s + b s^3 + c s^5, while the
//   singular vectors stay: the result is close to the nearest matrix with
//   orthonormal rows (or columns).
//   Muon: m <- mu m + g', u = g' + mu m (Nesterov) or m,
//   p <- p (1 - lr decay) - lr scale NS(u).
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "yl_internal.h"
#include "yl_muon.h"
#include "yume_c.h"

namespace yl {
namespace {

constexpr int kMaxItems = 64;    // matrices of one launch (their table is a kernel argument)
constexpr int kNormChunk = 16384;  // elements of one partial of a Frobenius norm
constexpr int kTile = 64;

struct Item {
  const float* src;   // NS: x; Muon: the gradient
  float* mom;         // Muon: momentum, contiguous
  float* dst;         // NS: y; Muon: the parameter
  long long lds, ldd;
  int rows, cols;
  float scale;
  int m, n;           // shorter and longer side
  float *x0, *x1, *a, *p;  // workspace: [m][n], [m][n], [m][m], [m][m]
  double* part;       // partial sums of squares
  int chunks;
};
struct Pack {
  Item it[kMaxItems];
  int start[kMaxItems + 1];  // blocks of the launch before each item
  int count;
};
struct Update {
  int muon, nesterov, sanitize;
  float mu, lr, decay, grad_scale, clip, eps;
  const float* norm;
};

__device__ __forceinline__ int find_item(const Pack& p, int block) {
  int k = 0;
  while (k + 1 < p.count && p.start[k + 1] <= block) ++k;
  return k;
}

__device__ __forceinline__ float clean(float g, const Update& u, float clipf) {
  float v = g * u.grad_scale;
  if (u.sanitize && !isfinite(v)) v = 0.f;
  return v * clipf;
}
__device__ __forceinline__ float clip_factor(const Update& u) {
  if (u.clip > 0.f && u.norm && *u.norm > u.clip) return u.clip / *u.norm;
  return 1.f;
}

// Sum over a block of 256 threads in a fixed order (valid in thread 0).
__device__ __forceinline__ double block_sum256(double s) {
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  double t = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < 8; ++w) t += red[w];
  return t;
}

// The momentum step and the partial sums of squares of u.
__global__ void ns_norm_kernel(const __grid_constant__ Pack p, const __grid_constant__ Update u) {
  const int k = find_item(p, blockIdx.x);
  const Item& it = p.it[k];
  const int chunk = blockIdx.x - p.start[k];
  const long long total = (long long)it.rows * it.cols;
  const long long lo = (long long)chunk * kNormChunk;
  const long long hi = min(total, lo + (long long)kNormChunk);
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  double s = 0.0;
  for (long long i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    float v;
    if (u.muon) {
      const float g = clean(it.src[i], u, clipf);
      const float m = u.mu * it.mom[i] + g;
      it.mom[i] = m;
      v = u.nesterov ? g + u.mu * m : m;
    } else {
      const long long r = i / it.cols;
      v = it.src[r * it.lds + (i - r * it.cols)];
    }
    s += (double)v * v;
  }
  s = block_sum256(s);
  if (threadIdx.x == 0) it.part[chunk] = s;
}

// part[block] = sum of squares of one chunk of scaled (and sanitized) gradients
__global__ void grad_square_kernel(const float* __restrict__ g, long long n, float scale,
                                   int sanitize, double* __restrict__ part) {
  const long long lo = blockIdx.x * (long long)kNormChunk;
  const long long hi = min(n, lo + (long long)kNormChunk);
  double s = 0.0;
  for (long long i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    float v = g[i] * scale;
    if (sanitize && !isfinite(v)) v = 0.f;
    s += (double)v * v;
  }
  s = block_sum256(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}
__global__ void grad_norm_final_kernel(const double* __restrict__ part, long long n, float* norm) {
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) s += part[i];
  s = block_sum256(s);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// X0 = u / (|u| + eps), transposed when the rows are the longer side.
__global__ void ns_scale_kernel(const __grid_constant__ Pack p, const __grid_constant__ Update u) {
  const int k = find_item(p, blockIdx.x);
  const Item& it = p.it[k];
  const int chunk = blockIdx.x - p.start[k];
  double s = 0.0;
  for (int c = 0; c < it.chunks; ++c) s += it.part[c];
  const float inv = (float)(1.0 / (sqrt(s) + (double)u.eps));
  const long long total = (long long)it.rows * it.cols;
  const long long lo = (long long)chunk * kNormChunk;
  const long long hi = min(total, lo + (long long)kNormChunk);
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  for (long long i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    const long long r = i / it.cols, c = i - r * it.cols;
    float v;
    if (u.muon) {
      v = it.mom[i];
      if (u.nesterov) v = clean(it.src[i], u, clipf) + u.mu * v;
    } else {
      v = it.src[r * it.lds + c];
    }
    it.x0[it.rows > it.cols ? c * it.n + r : i] = v * inv;
  }
}

enum { GRAM = 0, SQUARE = 1, UPDATE = 2 };

// One 64 x 64 tile of A = X X^T, P = a I + b A + c A A or X' = P X.
template <int MODE>
__global__ void __launch_bounds__(256)
    ns_product_kernel(const __grid_constant__ Pack p, float a, float b, float c, int flip) {
  const int k = find_item(p, blockIdx.x);
  const Item& it = p.it[k];
  const int m = it.m, N = MODE == UPDATE ? it.n : m, K = MODE == GRAM ? it.n : m;
  const int tn = (N + kTile - 1) / kTile;
  const int t = blockIdx.x - p.start[k];
  const int r0 = (t / tn) * kTile, c0 = (t % tn) * kTile;
  const float* x = flip ? it.x1 : it.x0;
  const float* L = MODE == GRAM ? x : MODE == SQUARE ? it.a : it.p;
  const float* R = MODE == SQUARE ? it.a : x;
  float* out = MODE == GRAM ? it.a : MODE == SQUARE ? it.p : (flip ? it.x0 : it.x1);
  const int ldl = MODE == GRAM ? it.n : m, ldr = MODE == SQUARE ? m : it.n;
  __shared__ float sl[16][kTile + 1], sr[16][kTile + 1];
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int e = threadIdx.x; e < 16 * kTile; e += 256) {
      const int kk = e % 16, r = e / 16;
      sl[kk][r] = (r0 + r < m && k0 + kk < K) ? L[(long long)(r0 + r) * ldl + k0 + kk] : 0.f;
      if (MODE == GRAM) {
        sr[kk][r] = (c0 + r < N && k0 + kk < K) ? R[(long long)(c0 + r) * ldr + k0 + kk] : 0.f;
      } else {
        const int cc = e % kTile, kr = e / kTile;
        sr[kr][cc] = (c0 + cc < N && k0 + kr < K) ? R[(long long)(k0 + kr) * ldr + c0 + cc] : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sl[kk][ty * 4 + i], sr[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + ty * 4 + i, cc = c0 + tx * 4 + j;
      if (r >= m || cc >= N) continue;
      const long long o = (long long)r * N + cc;
      out[o] = MODE == SQUARE ? (r == cc ? a : 0.f) + b * it.a[o] + c * acc[i][j] : acc[i][j];
    }
}

// y = X, or p <- p (1 - lr decay) - lr scale X.
__global__ void ns_finish_kernel(const __grid_constant__ Pack p, const __grid_constant__ Update u,
                                 int flip) {
  const int k = find_item(p, blockIdx.x);
  const Item& it = p.it[k];
  const int chunk = blockIdx.x - p.start[k];
  const float* x = flip ? it.x1 : it.x0;
  const long long total = (long long)it.rows * it.cols;
  const long long lo = (long long)chunk * kNormChunk;
  const long long hi = min(total, lo + (long long)kNormChunk);
  for (long long i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    const long long r = i / it.cols, c = i - r * it.cols;
    const float v = x[it.rows > it.cols ? c * it.n + r : i];
    if (u.muon) it.dst[i] = it.dst[i] * (1.f - u.lr * u.decay) - u.lr * it.scale * v;
    else it.dst[r * it.ldd + c] = v;
  }
}

// Sizes the items' workspaces, or (with a base address) places them; returns
// the bytes they take.
size_t place(Item* items, int count, char* ws) {
  ScratchCarver carve;
  for (int k = 0; k < count; ++k) {
    Item& it = items[k];
    it.m = std::min(it.rows, it.cols);
    it.n = std::max(it.rows, it.cols);
    it.chunks = (int)(((long long)it.rows * it.cols + kNormChunk - 1) / kNormChunk);
    const size_t mn = (size_t)it.m * it.n * 4, mm = (size_t)it.m * it.m * 4;
    it.x0 = (float*)(ws + carve.take(mn));
    it.x1 = (float*)(ws + carve.take(mn));
    it.a = (float*)(ws + carve.take(mm));
    it.p = (float*)(ws + carve.take(mm));
    it.part = (double*)(ws + carve.take(it.chunks * sizeof(double)));
  }
  return carve.offset;
}

yl_status run_pack(yl_ctx* ctx, Pack& p, const Update& u, int steps, const float* coeffs,
                   char* ws) {
  place(p.it, p.count, ws);
  auto starts = [&](auto blocks) {
    p.start[0] = 0;
    for (int k = 0; k < p.count; ++k) p.start[k + 1] = p.start[k] + blocks(p.it[k]);
    return (unsigned)p.start[p.count];
  };
  auto tiles = [](int v) { return (v + kTile - 1) / kTile; };
  unsigned grid = starts([](const Item& it) { return it.chunks; });
  ns_norm_kernel<<<grid, 256, 0, ctx->stream>>>(p, u);
  YL_TRY(check_launch("ns_norm_kernel"));
  ns_scale_kernel<<<grid, 256, 0, ctx->stream>>>(p, u);
  YL_TRY(check_launch("ns_scale_kernel"));
  int flip = 0;
  for (int s = 0; s < steps; ++s, flip ^= 1) {
    const float a = coeffs[3 * s], b = coeffs[3 * s + 1], c = coeffs[3 * s + 2];
    grid = starts([&](const Item& it) { return tiles(it.m) * tiles(it.m); });
    ns_product_kernel<GRAM><<<grid, 256, 0, ctx->stream>>>(p, a, b, c, flip);
    YL_TRY(check_launch("ns_product_kernel"));
    ns_product_kernel<SQUARE><<<grid, 256, 0, ctx->stream>>>(p, a, b, c, flip);
    YL_TRY(check_launch("ns_product_kernel"));
    grid = starts([&](const Item& it) { return tiles(it.m) * tiles(it.n); });
    ns_product_kernel<UPDATE><<<grid, 256, 0, ctx->stream>>>(p, a, b, c, flip);
    YL_TRY(check_launch("ns_product_kernel"));
  }
  grid = starts([](const Item& it) { return it.chunks; });
  ns_finish_kernel<<<grid, 256, 0, ctx->stream>>>(p, u, flip);
  return check_launch("ns_finish_kernel");
}

// All packs of a call, one after the other in the same workspace.
yl_status run_items(yl_ctx* ctx, std::vector<Item>& items, const Update& u, int steps,
                    const float* coeffs, char* ws) {
  for (size_t base = 0; base < items.size(); base += kMaxItems) {
    Pack p;
    p.count = (int)std::min<size_t>(kMaxItems, items.size() - base);
    std::copy_n(items.begin() + base, p.count, p.it);
    YL_TRY(run_pack(ctx, p, u, steps, coeffs, ws));
  }
  return YL_OK;
}
size_t items_bytes(std::vector<Item>& items) {
  size_t most = 0;
  for (size_t base = 0; base < items.size(); base += kMaxItems)
    most = std::max(most, place(items.data() + base,
                                (int)std::min<size_t>(kMaxItems, items.size() - base), nullptr));
  return most;
}

size_t norm_parts(long long n) { return (size_t)((n + kNormChunk - 1) / kNormChunk); }

constexpr float kQuintic[3] = {3.4445f, -4.7750f, 2.0315f};
constexpr int kMaxSteps = 32;
// Largest singular value the iteration may reach on the way.
constexpr double kMaxSigma = 4.0;

// The coefficients of every step, and whether they keep the singular values
// (at most 1 at the start) below kMaxSigma.
yl_status coefficients(const char* who, int steps, const float* given, float* out) {
  YL_CHECK(steps >= 0 && steps <= kMaxSteps, YL_ERR_INVALID, "%s: %d steps (0 to %d)", who, steps,
           kMaxSteps);
  double top = 1.0;
  for (int s = 0; s < steps; ++s) {
    const float* q = given ? given + 3 * s : kQuintic;
    for (int i = 0; i < 3; ++i) {
      YL_CHECK(std::isfinite(q[i]), YL_ERR_INVALID, "%s: coefficient %d of step %d is not finite",
               who, i, s);
      out[3 * s + i] = q[i];
    }
    // |p| on [0, top] is largest at its end or where p' = a + 3 b s^2 + 5 c s^4 = 0
    const double a = q[0], b = q[1], c = q[2];
    auto p = [&](double v) { return std::fabs(v * (a + v * v * (b + v * v * c))); };
    double next = p(top);
    auto at = [&](double sq) {
      if (sq > 0 && sq < top * top) next = std::max(next, p(std::sqrt(sq)));
    };
    if (c == 0.0) {
      if (b != 0.0) at(-a / (3 * b));
    } else {
      const double d = 9 * b * b - 20 * a * c;
      if (d >= 0) {
        at((-3 * b + std::sqrt(d)) / (10 * c));
        at((-3 * b - std::sqrt(d)) / (10 * c));
      }
    }
    const double inner = std::fabs(a) + std::fabs(b) * top * top + std::fabs(c) * top * top * top * top;
    YL_CHECK(next <= kMaxSigma && inner <= 1024.0, YL_ERR_UNSUPPORTED,
             "%s: the coefficients of step %d let singular values grow to %.3g (at most %.3g)", who,
             s, next, kMaxSigma);
    top = next;
  }
  return YL_OK;
}

yl_status check_shape(const char* who, int k, int rows, int cols) {
  YL_CHECK(rows >= 0 && cols >= 0 && rows <= kNsMaxSide && cols <= kNsMaxSide, YL_ERR_SHAPE,
           "%s: matrix %d is %d x %d (sides of 0 to %d)", who, k, rows, cols, kNsMaxSide);
  return YL_OK;
}

}  // namespace

bool rows_overlap(const float* a, long long lda, long long rows_a, long long cols_a,
                  const float* b, long long ldb, long long rows_b, long long cols_b) {
  if (!a || !b || rows_a <= 0 || rows_b <= 0 || cols_a <= 0 || cols_b <= 0) return false;
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + 4 * ((uintptr_t)(rows_a - 1) * lda + cols_a);
  const uintptr_t b1 = b0 + 4 * ((uintptr_t)(rows_b - 1) * ldb + cols_b);
  if (a1 <= b0 || b1 <= a0) return false;
  if (lda != ldb) return true;
  // columns of one buffer side by side?  (b - a) modulo the row stride
  long long d = ((long long)(b0 - a0) / 4) % lda;
  if (d < 0) d += lda;
  return !(d >= cols_a && d + cols_b <= lda);
}

yl_status newton_schulz(yl_ctx* ctx, const yl_ns_matrix* table, int count, int steps,
                        const float* coeffs, float eps) {
  const char* who = "yl_newton_schulz";
  float q[3 * kMaxSteps];
  YL_TRY(coefficients(who, steps, coeffs, q));
  YL_CHECK(eps >= 0.f, YL_ERR_INVALID, "%s: eps %g is negative or NaN", who, (double)eps);
  std::vector<Item> items;
  for (int k = 0; k < count; ++k) {
    const yl_ns_matrix& t = table[k];
    YL_TRY(check_shape(who, k, t.rows, t.cols));
    if (t.rows == 0 || t.cols == 0) continue;
    YL_CHECK(t.x && t.y, YL_ERR_INVALID, "%s: NULL pointer in matrix %d", who, k);
    YL_CHECK(t.ldx >= t.cols && t.ldy >= t.cols, YL_ERR_SHAPE,
             "%s: a row stride of matrix %d is smaller than its %d columns", who, k, t.cols);
    YL_CHECK(!((uintptr_t)t.x & 3) && !((uintptr_t)t.y & 3), YL_ERR_INVALID,
             "%s: a pointer of matrix %d is not a multiple of 4 bytes", who, k);
    Item it{};
    it.src = t.x, it.dst = t.y, it.lds = t.ldx, it.ldd = t.ldy, it.rows = t.rows, it.cols = t.cols;
    items.push_back(it);
  }
  for (size_t i = 0; i < items.size(); ++i)
    for (size_t j = 0; j < items.size(); ++j) {
      const Item &u = items[i], &v = items[j];
      if (i < j)
        YL_CHECK(!rows_overlap(u.dst, u.ldd, u.rows, u.cols, v.dst, v.ldd, v.rows, v.cols),
                 YL_ERR_INVALID, "%s: two results overlap", who);
      if (i == j && u.src == v.dst && u.lds == v.ldd) continue;  // in place
      YL_CHECK(!rows_overlap(u.src, u.lds, u.rows, u.cols, v.dst, v.ldd, v.rows, v.cols),
               YL_ERR_INVALID, "%s: a result overlaps an input", who);
    }
  if (items.empty()) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  Update u{};
  u.eps = eps;
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, items_bytes(items), &ws));
  YL_TRY(run_items(ctx, items, u, steps, q, ws));
  return work.done();
}

yl_status grad_norm(yl_ctx* ctx, const float* g, long long n, float grad_scale, int sanitize,
                    float* norm_out) {
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  const size_t parts = norm_parts(n);
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, parts * sizeof(double), &ws));
  if (parts) {
    grad_square_kernel<<<(unsigned)parts, 256, 0, ctx->stream>>>(g, n, grad_scale, sanitize,
                                                                 (double*)ws);
    YL_TRY(check_launch("grad_square_kernel"));
  }
  grad_norm_final_kernel<<<1, 256, 0, ctx->stream>>>((const double*)ws, (long long)parts, norm_out);
  YL_TRY(check_launch("grad_norm_final_kernel"));
  return work.done();
}

yl_status muon_multi(yl_ctx* ctx, const yl_muon_tensor* table, int count, const MuonStep& st,
                     const float* coeffs, const float* norm, float* norm_out) {
  const char* who = "yl_muon_multi";
  float q[3 * kMaxSteps];
  YL_TRY(coefficients(who, st.steps, coeffs, q));
  YL_CHECK(st.eps >= 0.f, YL_ERR_INVALID, "%s: eps %g is negative or NaN", who, (double)st.eps);
  std::vector<Item> items;
  for (int k = 0; k < count; ++k) {
    const yl_muon_tensor& t = table[k];
    YL_TRY(check_shape(who, k, t.rows, t.cols));
    if (t.rows == 0 || t.cols == 0) continue;
    YL_CHECK(t.param && t.grad && t.momentum, YL_ERR_INVALID, "%s: NULL pointer in matrix %d", who,
             k);
    YL_CHECK(!(((uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.momentum) & 3),
             YL_ERR_INVALID, "%s: a pointer of matrix %d is not a multiple of 4 bytes", who, k);
    Item it{};
    it.src = t.grad, it.mom = t.momentum, it.dst = t.param;
    it.lds = it.ldd = t.cols;
    it.rows = t.rows, it.cols = t.cols, it.scale = t.scale;
    items.push_back(it);
  }
  // each parameter and momentum is written once, and no gradient is
  struct Range { uintptr_t lo, hi; bool write; };
  std::vector<Range> r;
  for (const Item& it : items) {
    const uintptr_t bytes = (uintptr_t)4 * it.rows * it.cols;
    r.push_back({(uintptr_t)it.src, (uintptr_t)it.src + bytes, false});
    r.push_back({(uintptr_t)it.mom, (uintptr_t)it.mom + bytes, true});
    r.push_back({(uintptr_t)it.dst, (uintptr_t)it.dst + bytes, true});
  }
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
  uintptr_t end = 0, wend = 0;  // behind every range so far, and every written one
  for (const Range& x : r) {
    YL_CHECK(!(x.lo < wend || (x.write && x.lo < end)), YL_ERR_INVALID,
             "%s: a parameter or momentum overlaps another tensor of the table", who);
    end = std::max(end, x.hi);
    if (x.write) wend = std::max(wend, x.hi);
  }
  const bool measure = norm_out || (st.clip_max_norm > 0.f && !norm);
  if (items.empty() && !measure) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  size_t parts = 0;
  if (measure)
    for (const Item& it : items) parts += norm_parts((long long)it.rows * it.cols);
  ScratchCarver carve;
  const size_t o_norm = carve.take(sizeof(float)), o_parts = carve.take(parts * sizeof(double));
  const size_t o_items = carve.take(items_bytes(items));
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, carve.offset, &ws));
  if (measure) {
    double* part = (double*)(ws + o_parts);
    float* out = norm_out ? norm_out : (float*)(ws + o_norm);
    for (const Item& it : items) {
      const long long n = (long long)it.rows * it.cols;
      grad_square_kernel<<<(unsigned)norm_parts(n), 256, 0, ctx->stream>>>(it.src, n, st.grad_scale,
                                                                           st.sanitize, part);
      YL_TRY(check_launch("grad_square_kernel"));
      part += norm_parts(n);
    }
    grad_norm_final_kernel<<<1, 256, 0, ctx->stream>>>((const double*)(ws + o_parts),
                                                       (long long)parts, out);
    YL_TRY(check_launch("grad_norm_final_kernel"));
    if (!norm) norm = out;
  }
  Update u{};
  u.muon = 1, u.nesterov = st.nesterov, u.sanitize = st.sanitize;
  u.mu = st.momentum, u.lr = st.lr, u.decay = st.weight_decay, u.grad_scale = st.grad_scale;
  u.clip = st.clip_max_norm, u.eps = st.eps, u.norm = norm;
  YL_TRY(run_items(ctx, items, u, st.steps, q, ws + o_items));
  return work.done();
}

}  // namespace yl

using namespace yl;

extern "C" {

yl_status yl_newton_schulz(yl_ctx* ctx, const yl_ns_matrix* table, int count, int steps,
                           const float* coeffs, float eps) {
  YL_CHECK(ctx && (table || count == 0), YL_ERR_INVALID, "yl_newton_schulz: NULL argument");
  YL_CHECK(count >= 0, YL_ERR_INVALID, "yl_newton_schulz: negative matrix count");
  try {
    return newton_schulz(ctx, table, count, steps, coeffs, eps);
  } catch (const std::bad_alloc&) {
    return set_error(YL_ERR_OOM, "yl_newton_schulz: no host memory for %d matrices", count);
  }
}

yl_status yl_muon_multi(yl_ctx* ctx, const yl_muon_tensor* table, int count, float lr,
                        float momentum, int nesterov, float weight_decay, int steps,
                        const float* coeffs, float eps, float grad_scale, float clip_max_norm,
                        int sanitize, float* norm_out_dev) {
  YL_CHECK(ctx && (table || count == 0), YL_ERR_INVALID, "yl_muon_multi: NULL argument");
  YL_CHECK(count >= 0, YL_ERR_INVALID, "yl_muon_multi: negative matrix count");
  MuonStep st;
  st.lr = lr, st.momentum = momentum, st.nesterov = nesterov != 0, st.weight_decay = weight_decay;
  st.steps = steps, st.eps = eps, st.grad_scale = grad_scale, st.clip_max_norm = clip_max_norm;
  st.sanitize = sanitize != 0;
  try {
    return muon_multi(ctx, table, count, st, coeffs, nullptr, norm_out_dev);
  } catch (const std::bad_alloc&) {
    return set_error(YL_ERR_OOM, "yl_muon_multi: no host memory for %d matrices", count);
  }
}

}  // extern "C"
