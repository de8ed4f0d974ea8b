// yl_layernorm.cu -- LayerNorm over the last axis of [rows][cols] fp32,
// forward and backward.
//
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  r = 1 / sqrt(var + eps),
//   h = (x - mean) r,  y = h gamma + beta;
//   t = dy gamma,  dx = r (t - mean(t) - h mean(t h)) (+ addend),
//   dgamma = sum over rows of dy h,  dbeta = sum over rows of dy.
//
// Bound by HBM: 8 bytes an element forward, 12 backward (16 with an addend).
// A row is held in registers from its only read to its only write:
//   up to 1024 columns   a group of 4 to 32 lanes owns a row, several rows in
//                        flight per group where a row is short;
//   up to 16384 columns  a block of 256 to 1024 threads owns a row;
//   longer               a block walks the row from memory again for each pass.
// The mean of x - mean, which fp32 leaves not quite zero, is measured with the
// variance and taken off again, so that rows far from zero keep their accuracy.
// The column sums of the backward pass stay with the threads that own the columns
// (in registers, past 8192 columns in shared memory); after at most 64 rows they go
// to a block's partial row, and a second kernel adds the partial rows in double in a
// fixed order.
#include <algorithm>
#include <type_traits>

#include "yl_internal.h"
#include "yl_muon.h"
#include "yl_ptx.cuh"
#include "yume_c.h"

using namespace yl;

namespace {

constexpr int kSegRows = 64;  // rows a thread sums in fp32 before a partial is written
// Backward calls whose rows one block sees in so many turns run in that block
// alone: 32 x 512 in one kernel of 4 turns, not two kernels.
constexpr int kAloneTurns = 4;

// ---------------------------------------------------------------- row pieces
// Element e of a lane's PER elements is column (e / 4 * LANES + lane) * 4 + e % 4
// with 16-byte accesses and e * LANES + lane without.
template <int LANES, int PER, bool VEC>
struct Row {
  static constexpr int kCols = LANES * PER;
  static __device__ __forceinline__ int col(int e, int lane) {
    return VEC ? ((e >> 2) * LANES + lane) * 4 + (e & 3) : e * LANES + lane;
  }
  static __device__ __forceinline__ void load(const float* p, int cols, int lane, float (&v)[PER]) {
    if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < PER / 4; ++q) {
        const int c = (q * LANES + lane) * 4;
        const float4 f = c < cols ? __ldcs(reinterpret_cast<const float4*>(p + c))
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
        v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = col(e, lane) < cols ? p[col(e, lane)] : 0.f;
    }
  }
  static __device__ __forceinline__ void load_or(const float* p, float other, int cols, int lane,
                                                 float (&v)[PER]) {
    if (p) {
      if constexpr (VEC) {
#pragma unroll
        for (int q = 0; q < PER / 4; ++q) {
          const int c = (q * LANES + lane) * 4;
          const float4 f = c < cols ? __ldg(reinterpret_cast<const float4*>(p + c))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
          v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) v[e] = col(e, lane) < cols ? __ldg(p + col(e, lane)) : 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] = other;
    }
  }
  static __device__ __forceinline__ void store(float* p, int cols, int lane, const float (&v)[PER]) {
    if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < PER / 4; ++q) {
        const int c = (q * LANES + lane) * 4;
        if (c < cols)
          __stcs(reinterpret_cast<float4*>(p + c),
                 make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (col(e, lane) < cols) p[col(e, lane)] = v[e];
    }
  }
};

// Sums over the threads that own a row: a group of lanes, or a whole block.
template <int LANES>
struct Group {
  static __device__ __forceinline__ void sum(float& a, float*) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  static __device__ __forceinline__ void sum2(float& a, float& b, float*) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
};
template <int THREADS>
struct Block {
  static __device__ __forceinline__ void sum2(float& a, float& b, float* red) {
    Group<32>::sum2(a, b, nullptr);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      red[threadIdx.x >> 5] = a;
      red[32 + (threadIdx.x >> 5)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      a += red[w];
      b += red[32 + w];
    }
  }
  static __device__ __forceinline__ void sum(float& a, float* red) {
    float b = 0.f;
    sum2(a, b, red);
  }
};

// mean (rounded), what it is short of, and 1 / sqrt(var + eps).  A row whose sums pass
// fp32's range becomes NaN, as one with a NaN or an infinity does.  (A second look at
// such rows with the differences scaled down, in registers or from memory, cost all
// others: 25000 x 2047 forward 90 to 103 us, 6000 x 8192 backward 135 to 148.)
template <class Own, class R, int PER>
__device__ __forceinline__ void row_stats(const float (&x)[PER], int cols, int lane, float eps,
                                          float* red, float& m, float& e, float& rs) {
  const float inv = 1.f / cols;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) s += x[k];
  Own::sum(s, red);
  m = s * inv;
  float d1 = 0.f, d2 = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (R::col(k, lane) < cols) {
      const float d = x[k] - m;
      d1 += d;
      d2 = fmaf(d, d, d2);
    }
  Own::sum2(d1, d2, red);
  e = d1 * inv;
  rs = 1.f / sqrtf(fmaxf(fmaf(-e, e, d2 * inv), 0.f) + eps);
  if (!(d2 < INFINITY)) rs = NAN;
}

struct Fwd {
  const float* x;
  long long ldx, rows;
  int cols;
  float eps;
  const float *gamma, *beta;
  float* y;
  long long ldy;
  float *mean, *rstd;
};

// UNR rows of a group are read before the first is worked on.
template <int LANES, int PER, int UNR>
__global__ void __launch_bounds__(256) ln_fwd_group_kernel(const __grid_constant__ Fwd p) {
  using R = Row<LANES, PER, false>;
  const int lane = threadIdx.x % LANES;
  float ga[PER], be[PER];
  R::load_or(p.gamma, 1.f, p.cols, lane, ga);
  R::load_or(p.beta, 0.f, p.cols, lane, be);
  const long long per_block = (256 / LANES) * UNR;
  for (long long r0 = blockIdx.x * per_block; r0 < p.rows; r0 += gridDim.x * per_block) {
    const long long r = r0 + threadIdx.x / LANES;
    float x[UNR][PER];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const long long ru = min(r + u * (256 / LANES), p.rows - 1);  // every lane takes part
      R::load(p.x + ru * p.ldx, p.cols, lane, x[u]);
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const long long ru = r + u * (256 / LANES);
      float m, e, rs, y[PER];
      row_stats<Group<LANES>, R, PER>(x[u], p.cols, lane, p.eps, nullptr, m, e, rs);
#pragma unroll
      for (int k = 0; k < PER; ++k) y[k] = fmaf(((x[u][k] - m) - e) * rs, ga[k], be[k]);
      if (ru < p.rows) {
        R::store(p.y + ru * p.ldy, p.cols, lane, y);
        if (lane == 0) {
          if (p.mean) p.mean[ru] = m + e;
          if (p.rstd) p.rstd[ru] = rs;
        }
      }
    }
  }
}

template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS) ln_fwd_block_kernel(const __grid_constant__ Fwd p) {
  using R = Row<THREADS, PER, false>;
  __shared__ float red[64];
  const int lane = threadIdx.x;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    float x[PER], w[PER], m, e, rs;
    R::load(p.x + r * p.ldx, p.cols, lane, x);
    row_stats<Block<THREADS>, R, PER>(x, p.cols, lane, p.eps, red, m, e, rs);
    R::load_or(p.gamma, 1.f, p.cols, lane, w);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = ((x[k] - m) - e) * rs * w[k];
    R::load_or(p.beta, 0.f, p.cols, lane, w);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] += w[k];
    R::store(p.y + r * p.ldy, p.cols, lane, x);
    if (lane == 0) {
      if (p.mean) p.mean[r] = m + e;
      if (p.rstd) p.rstd[r] = rs;
    }
  }
}

// Rows of 16-byte aligned pieces.  Every thread copies its own pieces of the rows
// it will work on next into its own slots of a shared-memory ring (cp.async, D
// rows deep), so that reads keep running through the reductions without holding
// registers, and no thread waits for another's copy.
template <int N>
__device__ __forceinline__ void cp_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int THREADS, int LANES, int PER, int ARRAYS, int D>
struct Ring {
  static constexpr int kBytes = D * ARRAYS * (PER / 4) * THREADS * 16;
  static __device__ __forceinline__ uint8_t* slot(uint8_t* smem, int d, int a, int q) {
    return smem + (((d * ARRAYS + a) * (PER / 4) + q) * THREADS + threadIdx.x) * 16;
  }
  static __device__ __forceinline__ void fetch(uint8_t* smem, int d, int a, const float* row,
                                               int cols, int lane) {
#pragma unroll
    for (int q = 0; q < PER / 4; ++q) {
      const int c = (q * LANES + lane) * 4;
      cp_async_16(smem_u32(slot(smem, d, a, q)), c < cols ? row + c : row, c < cols);
    }
  }
  static __device__ __forceinline__ void take(uint8_t* smem, int d, int a, float (&v)[PER]) {
#pragma unroll
    for (int q = 0; q < PER / 4; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(slot(smem, d, a, q));
      v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
    }
  }
};

// Owner of a row: a group of LANES <= 32 lanes, or the whole block.
template <int THREADS, int LANES>
using Own = std::conditional_t<LANES <= 32, Group<LANES>, Block<THREADS>>;

template <int THREADS, int LANES, int PER, int D>
__global__ void __launch_bounds__(THREADS) ln_fwd_ring_kernel(const __grid_constant__ Fwd p) {
  using R = Row<LANES, PER, true>;
  using Q = Ring<THREADS, LANES, PER, 1, D>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[64];
  constexpr int G = THREADS / LANES;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const long long stride = (long long)gridDim.x * G;
  const long long iters = (p.rows + stride - 1) / stride;
  const long long first = (long long)blockIdx.x * G + grp;
  auto fetch = [&](long long it) {
    const long long r = min(first + it * stride, p.rows - 1);  // every lane takes part
    if (it < iters) Q::fetch(ring, (int)(it % D), 0, p.x + r * p.ldx, p.cols, lane);
    cp_commit();
  };
  for (int d = 0; d < D - 1; ++d) fetch(d);
  constexpr bool kKeep = PER <= 16;  // gamma and beta stay in registers
  float ga[PER], be[PER];
  if (kKeep) {
    R::load_or(p.gamma, 1.f, p.cols, lane, ga);
    R::load_or(p.beta, 0.f, p.cols, lane, be);
  }
  for (long long it = 0; it < iters; ++it) {
    fetch(it + D - 1);
    cp_wait_group<D - 1>();
    float x[PER], m, e, rs;
    Q::take(ring, (int)(it % D), 0, x);
    row_stats<Own<THREADS, LANES>, R, PER>(x, p.cols, lane, p.eps, red, m, e, rs);
    if (!kKeep) R::load_or(p.gamma, 1.f, p.cols, lane, ga);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = ((x[k] - m) - e) * rs * ga[k];
    if (!kKeep) R::load_or(p.beta, 0.f, p.cols, lane, be);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] += be[k];
    const long long r = first + it * stride;
    if (r < p.rows) {
      R::store(p.y + r * p.ldy, p.cols, lane, x);
      if (lane == 0) {
        if (p.mean) p.mean[r] = m + e;
        if (p.rstd) p.rstd[r] = rs;
      }
    }
  }
}

struct Bwd {
  const float *x, *dy;
  long long ldx, lddy, rows;
  int cols;
  float eps;
  const float *gamma, *mean, *rstd, *addend;
  long long ldadd;
  float* dx;
  long long lddx;
  // where column sums go: partial rows [partial][2][cols], or straight to dgamma
  // and dbeta (either may be null) when one block sees all rows
  float *part, *dgamma, *dbeta;
  __device__ bool sums() const { return part || dgamma || dbeta; }
  __device__ float* out_gamma(long long k) const { return part ? part + 2 * k * cols : dgamma; }
  __device__ float* out_beta(long long k) const {
    return part ? part + (2 * k + 1) * cols : dbeta;
  }
};

// dx of one row, and its share of the column sums.
// Add puts the addend's elements into an array.
template <class Own, class R, int PER, class Add>
__device__ __forceinline__ void bwd_row(const Bwd& p, long long r, bool valid, int lane,
                                        const float (&x)[PER], const float (&dy)[PER],
                                        const float (&ga)[PER], float m, float rs,
                                        float (&dg)[PER], float (&db)[PER], float* red, Add add) {
  // t rounded as in its mean, so that a row of one column gives exactly zero (in
  // all sizes that costs 10% of 16384 x 4096)
  constexpr bool kFew = R::kCols <= 16;
  float e = 0.f;
  if (!p.mean) row_stats<Own, R, PER>(x, p.cols, lane, p.eps, red, m, e, rs);
  float h[PER], s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    h[k] = R::col(k, lane) < p.cols ? ((x[k] - m) - e) * rs : 0.f;
    const float t = kFew ? __fmul_rn(dy[k], ga[k]) : dy[k] * ga[k];
    s1 += t;
    s2 = fmaf(t, h[k], s2);
  }
  if (p.dx) {
    Own::sum2(s1, s2, red);
    const float inv = 1.f / p.cols;
    s1 *= inv;
    s2 *= inv;
  }
  if (!valid) return;
  if (p.sums()) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      dg[k] = fmaf(dy[k], h[k], dg[k]);
      db[k] += dy[k];
    }
  }
  if (p.dx) {
    float out[PER];
    if (p.addend) add(out);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const float t = kFew ? __fmul_rn(dy[k], ga[k]) - s1 : fmaf(dy[k], ga[k], -s1);
      const float v = rs * (t - h[k] * s2);
      out[k] = p.addend ? out[k] + v : v;
    }
    R::store(p.dx + r * p.lddx, p.cols, lane, out);
  }
}

// A block adds its groups' column sums in order and writes a partial row; in double
// where the groups are many and the columns too few to average the roundings.
template <int LANES>
using GroupSum = std::conditional_t<LANES <= 8, double, float>;
template <int THREADS, int LANES, int PER, class R>
__device__ __forceinline__ void flush_groups(const Bwd& p, long long part, int lane, int grp,
                                             float (&dg)[PER], float (&db)[PER],
                                             GroupSum<LANES>* sums) {
  constexpr int CAP = LANES * PER;
  for (int g = 0; g < THREADS / LANES; ++g) {
    __syncthreads();
    if (grp == g) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = R::col(k, lane);
        sums[c] = g ? sums[c] + dg[k] : dg[k];
        sums[CAP + c] = g ? sums[CAP + c] + db[k] : db[k];
      }
    }
  }
  __syncthreads();
  float *og = p.out_gamma(part), *ob = p.out_beta(part);
  for (int c = threadIdx.x; c < p.cols; c += THREADS) {
    if (og) og[c] = (float)sums[c];
    if (ob) ob[c] = (float)sums[CAP + c];
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
}

template <int THREADS, int LANES, int PER, int D, int MIN_BLOCKS>
__global__ void __launch_bounds__(THREADS, MIN_BLOCKS) ln_bwd_ring_kernel(const __grid_constant__ Bwd p) {
  using R = Row<LANES, PER, true>;
  using Q = Ring<THREADS, LANES, PER, 3, D>;
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr bool kBlock = LANES > 32;
  __shared__ float red[kBlock ? 64 : 1];
  __shared__ GroupSum<LANES> sums[kBlock ? 1 : 2 * LANES * PER];
  constexpr int G = THREADS / LANES;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const long long stride = (long long)gridDim.x * G;
  const long long iters = (p.rows + stride - 1) / stride;
  const long long first = (long long)blockIdx.x * G + grp;
  auto fetch = [&](long long it) {
    const long long r = min(first + it * stride, p.rows - 1);  // every lane takes part
    if (it < iters) {
      const int d = (int)(it % D);
      Q::fetch(ring, d, 0, p.x + r * p.ldx, p.cols, lane);
      Q::fetch(ring, d, 1, p.dy + r * p.lddy, p.cols, lane);
      if (p.addend) Q::fetch(ring, d, 2, p.addend + r * p.ldadd, p.cols, lane);
    }
    cp_commit();
  };
  for (int d = 0; d < D - 1; ++d) fetch(d);
  float ga[PER], dg[PER], db[PER];
  R::load_or(p.gamma, 1.f, p.cols, lane, ga);
#pragma unroll
  for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
  long long part = blockIdx.x;
  int held = 0;
  for (long long it = 0; it < iters; ++it) {
    const long long r = first + it * stride, rc = min(r, p.rows - 1);
    const float m = p.mean ? __ldg(p.mean + rc) : 0.f, rs = p.mean ? __ldg(p.rstd + rc) : 0.f;
    fetch(it + D - 1);
    cp_wait_group<D - 1>();
    const int d = (int)(it % D);
    float x[PER], dy[PER];
    Q::take(ring, d, 0, x);
    Q::take(ring, d, 1, dy);
    bwd_row<Own<THREADS, LANES>, R, PER>(p, r, r < p.rows, lane, x, dy, ga, m, rs, dg, db, red,
                                         [&](float(&o)[PER]) { Q::take(ring, d, 2, o); });
    ++held;
    if (p.sums() && (held == kSegRows || it + 1 == iters)) {
      if constexpr (kBlock) {
        if (float* og = p.out_gamma(part)) R::store(og, p.cols, lane, dg);
        if (float* ob = p.out_beta(part)) R::store(ob, p.cols, lane, db);
#pragma unroll
        for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
      } else {
        flush_groups<THREADS, LANES, PER, R>(p, part, lane, grp, dg, db, sums);
      }
      part += gridDim.x;
      held = 0;
    }
  }
}

// Groups take rows in turns; every kSegRows rows of a group the block adds its
// groups' sums in order and writes a partial row.
template <int LANES, int PER, int UNR>
__global__ void __launch_bounds__(256) ln_bwd_group_kernel(const __grid_constant__ Bwd p) {
  using R = Row<LANES, PER, false>;
  constexpr int G = 256 / LANES;
  __shared__ GroupSum<LANES> sums[2 * LANES * PER];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  float ga[PER], dg[PER], db[PER];
  R::load_or(p.gamma, 1.f, p.cols, lane, ga);
#pragma unroll
  for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
  const long long stride = (long long)gridDim.x * G * UNR;
  const long long iters = (p.rows + stride - 1) / stride;
  long long part = blockIdx.x;
  int held = 0;
  for (long long it = 0; it < iters; ++it) {
    const long long r0 = it * stride + (long long)blockIdx.x * G * UNR + grp;
    float x[UNR][PER], dy[UNR][PER], m[UNR], rs[UNR];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const long long r = min(r0 + u * G, p.rows - 1);  // every lane takes part
      R::load(p.x + r * p.ldx, p.cols, lane, x[u]);
      R::load(p.dy + r * p.lddy, p.cols, lane, dy[u]);
      m[u] = p.mean ? __ldg(p.mean + r) : 0.f;
      rs[u] = p.mean ? __ldg(p.rstd + r) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u)
      bwd_row<Group<LANES>, R, PER>(p, r0 + u * G, r0 + u * G < p.rows, lane, x[u], dy[u], ga, m[u],
                                    rs[u], dg, db, nullptr, [&](float(&o)[PER]) {
                                      R::load(p.addend + (r0 + u * G) * p.ldadd, p.cols, lane, o);
                                    });
    held += UNR;
    if (p.sums() && (held + UNR > kSegRows || it + 1 == iters)) {
      flush_groups<256, LANES, PER, R>(p, part, lane, grp, dg, db, sums);
      part += gridDim.x;
      held = 0;
    }
  }
}

template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS) ln_bwd_block_kernel(const __grid_constant__ Bwd p) {
  using R = Row<THREADS, PER, false>;
  __shared__ float red[64];
  const int lane = threadIdx.x;
  float ga[PER], dg[PER], db[PER];
  R::load_or(p.gamma, 1.f, p.cols, lane, ga);
#pragma unroll
  for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
  const long long iters = (p.rows + gridDim.x - 1) / gridDim.x;
  long long part = blockIdx.x;
  int held = 0;
  for (long long it = 0; it < iters; ++it) {
    const long long r = it * gridDim.x + blockIdx.x;
    if (r < p.rows) {
      float x[PER], dy[PER];
      R::load(p.x + r * p.ldx, p.cols, lane, x);
      R::load(p.dy + r * p.lddy, p.cols, lane, dy);
      const float m = p.mean ? __ldg(p.mean + r) : 0.f, rs = p.mean ? __ldg(p.rstd + r) : 0.f;
      bwd_row<Block<THREADS>, R, PER>(
          p, r, true, lane, x, dy, ga, m, rs, dg, db, red,
          [&](float(&o)[PER]) { R::load(p.addend + r * p.ldadd, p.cols, lane, o); });
    }
    ++held;
    if (p.sums() && (held == kSegRows || it + 1 == iters)) {
      if (float* og = p.out_gamma(part)) R::store(og, p.cols, lane, dg);
      if (float* ob = p.out_beta(part)) R::store(ob, p.cols, lane, db);
#pragma unroll
      for (int k = 0; k < PER; ++k) dg[k] = db[k] = 0.f;
      part += gridDim.x;
      held = 0;
    }
  }
}

// Rows of more columns than the column sums leave registers for: those are in
// shared memory, each thread's own columns.
constexpr int kWideThreads = 1024, kWidePer = 16;
constexpr int kWideBytes = 2 * kWideThreads * kWidePer * (int)sizeof(float);

template <bool VEC>
__global__ void __launch_bounds__(kWideThreads) ln_bwd_wide_kernel(const __grid_constant__ Bwd p) {
  using R = Row<kWideThreads, kWidePer, VEC>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[64];
  const int lane = threadIdx.x;
  float* sums = reinterpret_cast<float*>(ring) + lane;  // [2][element][thread]
  constexpr int kBeta = kWidePer * kWideThreads;
#pragma unroll
  for (int k = 0; k < kWidePer; ++k) sums[k * kWideThreads] = sums[kBeta + k * kWideThreads] = 0.f;
  const long long iters = (p.rows + gridDim.x - 1) / gridDim.x;
  long long part = blockIdx.x;
  int held = 0;
  for (long long it = 0; it < iters; ++it) {
    const long long r = it * gridDim.x + blockIdx.x;
    if (r < p.rows) {
      float x[kWidePer], dy[kWidePer], w[kWidePer];
      R::load(p.x + r * p.ldx, p.cols, lane, x);
      R::load(p.dy + r * p.lddy, p.cols, lane, dy);
      float m = p.mean ? __ldg(p.mean + r) : 0.f, rs = p.mean ? __ldg(p.rstd + r) : 0.f, e = 0.f;
      if (!p.mean)
        row_stats<Block<kWideThreads>, R, kWidePer>(x, p.cols, lane, p.eps, red, m, e, rs);
      R::load_or(p.gamma, 1.f, p.cols, lane, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < kWidePer; ++k) {
        x[k] = R::col(k, lane) < p.cols ? ((x[k] - m) - e) * rs : 0.f;
        if (p.sums()) {
          sums[k * kWideThreads] = fmaf(dy[k], x[k], sums[k * kWideThreads]);
          sums[kBeta + k * kWideThreads] += dy[k];
        }
        dy[k] *= w[k];
        s1 += dy[k];
        s2 = fmaf(dy[k], x[k], s2);
      }
      if (p.dx) {
        if (p.addend) R::load(p.addend + r * p.ldadd, p.cols, lane, w);
        Block<kWideThreads>::sum2(s1, s2, red);
        const float inv = 1.f / p.cols;
        s1 *= inv;
        s2 *= inv;
#pragma unroll
        for (int k = 0; k < kWidePer; ++k) {
          const float v = rs * ((dy[k] - s1) - x[k] * s2);
          w[k] = p.addend ? w[k] + v : v;
        }
        R::store(p.dx + r * p.lddx, p.cols, lane, w);
      }
    }
    ++held;
    if (p.sums() && (held == kSegRows || it + 1 == iters)) {
      float *og = p.out_gamma(part), *ob = p.out_beta(part);
#pragma unroll
      for (int k = 0; k < kWidePer; ++k) {
        const int c = R::col(k, lane);
        if (c < p.cols) {
          if (og) og[c] = sums[k * kWideThreads];
          if (ob) ob[c] = sums[kBeta + k * kWideThreads];
        }
        sums[k * kWideThreads] = sums[kBeta + k * kWideThreads] = 0.f;
      }
      part += gridDim.x;
      held = 0;
    }
  }
}

// Column sums of the partial rows, 32 columns by 32 shares of the rows a block;
// blockIdx.y 0: dgamma, 1: dbeta.
__global__ void __launch_bounds__(1024)
    ln_bwd_columns_kernel(const float* __restrict__ part, long long parts, int cols,
                          float* __restrict__ dgamma, float* __restrict__ dbeta) {
  float* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  __shared__ double sums[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  double s = 0.0;
  if (c < cols) {
    const float* p = part + (long long)blockIdx.y * cols + c;
#pragma unroll 4
    for (long long k = share; k < parts; k += 32) s += (double)__ldg(p + 2 * k * cols);
  }
  sums[share][threadIdx.x & 31] = s;
  __syncthreads();
  // warp w adds the 32 shares of column w by a fixed tree
  double v = sums[threadIdx.x & 31][share];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int cw = blockIdx.x * 32 + share;
  if ((threadIdx.x & 31) == 0 && cw < cols) out[cw] = (float)v;
}

// ---------------------------------------------------------------- longer rows
// A thread adds up any number of elements here, so the row's sums are in double.
constexpr int kLong = 1024;

__device__ __forceinline__ void long_sum2(double& a, double& b, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = a;
    red[32 + (threadIdx.x >> 5)] = b;
  }
  __syncthreads();
  a = b = 0.0;
  for (int w = 0; w < kLong / 32; ++w) {
    a += red[w];
    b += red[32 + w];
  }
}

__device__ __forceinline__ void long_stats(const float* x, int cols, float eps, double* red,
                                           float& m, float& e, float& rs) {
  double s = 0.0, s2 = 0.0;
  for (int c = threadIdx.x; c < cols; c += kLong) s += (double)x[c];
  long_sum2(s, s2, red);
  m = (float)(s / cols);
  s = s2 = 0.0;
  for (int c = threadIdx.x; c < cols; c += kLong) {
    const float d = x[c] - m;
    s += (double)d;
    s2 += (double)d * d;
  }
  long_sum2(s, s2, red);
  s /= cols;
  s2 = s2 / cols - s * s;
  e = (float)s;
  rs = (float)(1.0 / sqrt((s2 < 0.0 ? 0.0 : s2) + (double)eps));
  if (!(s2 < INFINITY)) rs = NAN;  // a NaN, an infinity or a difference past fp32's range
}

__global__ void __launch_bounds__(kLong) ln_fwd_long_kernel(const __grid_constant__ Fwd p) {
  __shared__ double red[64];
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const float* x = p.x + r * p.ldx;
    float m, e, rs;
    long_stats(x, p.cols, p.eps, red, m, e, rs);
    for (int c = threadIdx.x; c < p.cols; c += kLong)
      p.y[r * p.ldy + c] = fmaf(((x[c] - m) - e) * rs, p.gamma ? p.gamma[c] : 1.f,
                                p.beta ? p.beta[c] : 0.f);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = m + e;
      if (p.rstd) p.rstd[r] = rs;
    }
  }
}

// A block adds each of its rows into its own partial row in memory; kSegRows
// rows at most, as in registers.
__global__ void __launch_bounds__(kLong) ln_bwd_long_kernel(const __grid_constant__ Bwd p) {
  __shared__ double red[64];
  const long long per = (p.rows + gridDim.x - 1) / gridDim.x;
  for (long long it = 0; it < per; ++it) {
    const long long r = it * gridDim.x + blockIdx.x;
    const long long part = (it / kSegRows) * gridDim.x + blockIdx.x;
    float* pg = p.part ? p.part + 2 * part * p.cols : nullptr;
    const bool first = it % kSegRows == 0;
    if (r >= p.rows) {
      if (pg && first)  // a partial row without rows
        for (long long c = threadIdx.x; c < 2LL * p.cols; c += kLong) pg[c] = 0.f;
      continue;
    }
    const float *x = p.x + r * p.ldx, *dy = p.dy + r * p.lddy;
    float m, e = 0.f, rs;
    if (p.mean) m = p.mean[r], rs = p.rstd[r];
    else long_stats(x, p.cols, p.eps, red, m, e, rs);
    double s1 = 0.0, s2 = 0.0;
    for (int c = threadIdx.x; c < p.cols; c += kLong) {
      const float d = dy[c], h = ((x[c] - m) - e) * rs, 
                  t = __fmul_rn(d, p.gamma ? p.gamma[c] : 1.f);
      s1 += (double)t;
      s2 += (double)t * h;
      if (pg) {
        pg[c] = first ? d * h : fmaf(d, h, pg[c]);
        pg[p.cols + c] = first ? d : pg[p.cols + c] + d;
      }
    }
    if (!p.dx) continue;
    long_sum2(s1, s2, red);
    const float c1 = (float)(s1 / p.cols), c2 = (float)(s2 / p.cols);
    for (int c = threadIdx.x; c < p.cols; c += kLong) {
      const float h = ((x[c] - m) - e) * rs;
      float v = rs * ((__fmul_rn(dy[c], p.gamma ? p.gamma[c] : 1.f) - c1) - h * c2);
      if (p.addend) v += p.addend[r * p.ldadd + c];
      p.dx[r * p.lddx + c] = v;
    }
  }
}

// ---------------------------------------------------------------- dispatch
// A row's owner by its length: f(kernel, threads, rows a block takes at a time,
// rows of those that one thread sees, bytes of its ring).
template <int THREADS, int LANES, int PER, int D, class F>
auto fwd_ring(F f) {
  return f(ln_fwd_ring_kernel<THREADS, LANES, PER, D>, THREADS, THREADS / LANES, 1,
           Ring<THREADS, LANES, PER, 1, D>::kBytes);
}
template <class F>
auto fwd_aligned(int cols, F f) {
  if (cols <= 16) return fwd_ring<256, 4, 4, 4>(f);
  if (cols <= 32) return fwd_ring<256, 4, 8, 4>(f);
  if (cols <= 64) return fwd_ring<256, 4, 16, 3>(f);
  if (cols <= 128) return fwd_ring<256, 8, 16, 3>(f);
  if (cols <= 256) return fwd_ring<256, 16, 16, 3>(f);
  if (cols <= 512) return fwd_ring<256, 32, 16, 3>(f);
  if (cols <= 1024) return fwd_ring<256, 32, 32, 2>(f);
  if (cols <= 2048) return fwd_ring<256, 256, 8, 3>(f);
  if (cols <= 4096) return fwd_ring<512, 512, 8, 3>(f);
  if (cols <= 8192) return fwd_ring<1024, 1024, 8, 3>(f);
  if (cols <= 16384) return fwd_ring<1024, 1024, 16, 2>(f);
  return f(ln_fwd_long_kernel, kLong, 1, 1, 0);
}
template <class F>
auto fwd_plain(int cols, F f) {
  if (cols <= 16) return f(ln_fwd_group_kernel<4, 4, 2>, 256, 128, 2, 0);
  if (cols <= 32) return f(ln_fwd_group_kernel<8, 4, 4>, 256, 128, 4, 0);
  if (cols <= 64) return f(ln_fwd_group_kernel<16, 4, 4>, 256, 64, 4, 0);
  if (cols <= 128) return f(ln_fwd_group_kernel<32, 4, 4>, 256, 32, 4, 0);
  if (cols <= 256) return f(ln_fwd_group_kernel<32, 8, 2>, 256, 16, 2, 0);
  if (cols <= 512) return f(ln_fwd_group_kernel<32, 16, 1>, 256, 8, 1, 0);
  if (cols <= 1024) return f(ln_fwd_group_kernel<32, 32, 1>, 256, 8, 1, 0);
  if (cols <= 2048) return f(ln_fwd_block_kernel<256, 8>, 256, 1, 1, 0);
  if (cols <= 4096) return f(ln_fwd_block_kernel<512, 8>, 512, 1, 1, 0);
  if (cols <= 8192) return f(ln_fwd_block_kernel<1024, 8>, 1024, 1, 1, 0);
  if (cols <= 16384) return f(ln_fwd_block_kernel<1024, 16>, 1024, 1, 1, 0);
  return f(ln_fwd_long_kernel, kLong, 1, 1, 0);
}
template <int THREADS, int LANES, int PER, int D, int MIN_BLOCKS, class F>
auto bwd_ring(F f) {
  return f(ln_bwd_ring_kernel<THREADS, LANES, PER, D, MIN_BLOCKS>, THREADS, THREADS / LANES, 1,
           Ring<THREADS, LANES, PER, 3, D>::kBytes);
}
template <class F>
auto bwd_aligned(int cols, F f) {
  if (cols <= 16) return bwd_ring<256, 4, 4, 3, 4>(f);
  if (cols <= 32) return bwd_ring<256, 4, 8, 2, 3>(f);
  if (cols <= 64) return bwd_ring<256, 8, 8, 2, 3>(f);
  if (cols <= 128) return bwd_ring<256, 16, 8, 2, 3>(f);
  if (cols <= 256) return bwd_ring<256, 32, 8, 2, 3>(f);
  if (cols <= 512) return bwd_ring<256, 32, 16, 2, 2>(f);
  if (cols <= 1024) return bwd_ring<256, 256, 4, 3, 4>(f);
  if (cols <= 2048) return bwd_ring<256, 256, 8, 2, 3>(f);
  if (cols <= 4096) return bwd_ring<512, 512, 8, 2, 2>(f);
  if (cols <= 8192) return bwd_ring<1024, 1024, 8, 2, 1>(f);
  if (cols <= 16384) return f(ln_bwd_wide_kernel<true>, kWideThreads, 1, 1, kWideBytes);
  return f(ln_bwd_long_kernel, kLong, 1, 1, 0);
}
template <class F>
auto bwd_plain(int cols, F f) {
  if (cols <= 16) return f(ln_bwd_group_kernel<4, 4, 2>, 256, 128, 2, 0);
  if (cols <= 32) return f(ln_bwd_group_kernel<8, 4, 2>, 256, 64, 2, 0);
  if (cols <= 64) return f(ln_bwd_group_kernel<16, 4, 2>, 256, 32, 2, 0);
  if (cols <= 128) return f(ln_bwd_group_kernel<32, 4, 2>, 256, 16, 2, 0);
  if (cols <= 256) return f(ln_bwd_group_kernel<32, 8, 2>, 256, 16, 2, 0);
  if (cols <= 512) return f(ln_bwd_group_kernel<32, 16, 1>, 256, 8, 1, 0);
  if (cols <= 1024) return f(ln_bwd_block_kernel<256, 4>, 256, 1, 1, 0);
  if (cols <= 2048) return f(ln_bwd_block_kernel<256, 8>, 256, 1, 1, 0);
  if (cols <= 4096) return f(ln_bwd_block_kernel<512, 8>, 512, 1, 1, 0);
  if (cols <= 8192) return f(ln_bwd_block_kernel<1024, 8>, 1024, 1, 1, 0);
  if (cols <= 16384) return f(ln_bwd_wide_kernel<false>, kWideThreads, 1, 1, kWideBytes);
  return f(ln_bwd_long_kernel, kLong, 1, 1, 0);
}

// Limits a grid to the kernel's resident blocks on the whole device.
template <class K>
yl_status resident(yl_ctx* ctx, K kernel, int threads, int smem, long long* blocks) {
  if (smem > 40 * 1024)
    YL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (*blocks <= ctx->num_sms) return YL_OK;
  int per = 0;
  YL_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem));
  *blocks = std::min(*blocks, (long long)std::max(per, 1) * ctx->num_sms);
  return YL_OK;
}

constexpr int kMaxCols = 1 << 29;  // column indexes and twice their number stay ints

bool aligned4(const void* p) { return ((uintptr_t)p & 3) == 0; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// An argument of a call: rows of cols floats at a row stride of ld.
struct Span {
  const float* p;
  long long ld, rows, cols;
};
// Whether one of the first `outs` spans shares an element with any other span;
// in_place: the two of this pair may be one and the same.
bool results_overlap(const Span* s, int outs, int count, int in_place_out, int in_place_in) {
  for (int i = 0; i < outs; ++i)
    for (int j = i + 1; j < count; ++j) {
      if (i == in_place_out && j == in_place_in && s[i].p == s[j].p && s[i].ld == s[j].ld) continue;
      if (rows_overlap(s[i].p, s[i].ld, s[i].rows, s[i].cols, s[j].p, s[j].ld, s[j].rows, s[j].cols))
        return true;
    }
  return false;
}

yl_status check_ln(yl_ctx* ctx, const char* who, long long rows, int cols, float eps) {
  YL_CHECK(ctx, YL_ERR_INVALID, "%s: ctx is NULL", who);
  YL_CHECK(rows >= 0 && cols >= 1 && cols <= kMaxCols, YL_ERR_SHAPE,
           "%s: %lld rows of %d columns (1 to %d)", who, rows, cols, kMaxCols);
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
  const Span spans[] = {{y, ldy, rows, cols},     {mean_out, rows, 1, rows}, {rstd_out, rows, 1, rows},
                        {x, ldx, rows, cols},     {gamma, cols, 1, cols},    {beta, cols, 1, cols}};
  YL_CHECK(!results_overlap(spans, 3, 6, 0, 3), YL_ERR_INVALID,
           "yl_layernorm_fwd: a result overlaps another argument");
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  const Fwd p{x, ldx, rows, cols, eps, gamma, beta, y, ldy, mean_out, rstd_out};
  const bool vec = aligned16(x) && aligned16(y) && aligned16(gamma) && aligned16(beta) &&
                   ((ldx | ldy | cols) & 3) == 0;
  auto launch = [&](auto kernel, int threads, int rows_a_block, int, int smem) -> yl_status {
    long long blocks = (rows + rows_a_block - 1) / rows_a_block;
    YL_TRY(resident(ctx, kernel, threads, smem, &blocks));
    kernel<<<(unsigned)blocks, threads, smem, ctx->stream>>>(p);
    return check_launch("ln_fwd_kernel");
  };
  return vec ? fwd_aligned(cols, launch) : fwd_plain(cols, launch);
}

yl_status yl_layernorm_bwd(yl_ctx* ctx, const float* x, long long ldx, const float* dy,
                           long long lddy, long long rows, int cols, float eps, const float* gamma,
                           const float* mean, const float* rstd, const float* addend,
                           long long ldadd, float* dx, long long lddx, float* dgamma,
                           float* dbeta) {
  YL_TRY(check_ln(ctx, "yl_layernorm_bwd", rows, cols, eps));
  YL_CHECK((mean == nullptr) == (rstd == nullptr), YL_ERR_INVALID,
           "yl_layernorm_bwd: mean and rstd are given together or not at all");
  YL_CHECK(aligned4(x) && aligned4(dy) && aligned4(gamma) && aligned4(mean) && aligned4(rstd) &&
               aligned4(addend) && aligned4(dx) && aligned4(dgamma) && aligned4(dbeta),
           YL_ERR_INVALID, "yl_layernorm_bwd: a pointer is not a multiple of 4 bytes");
  if (rows == 0) {
    DeviceGuard dev(ctx->device);
    YL_CUDA(dev.status());
    if (dgamma) YL_CUDA(cudaMemsetAsync(dgamma, 0, cols * sizeof(float), ctx->stream));
    if (dbeta) YL_CUDA(cudaMemsetAsync(dbeta, 0, cols * sizeof(float), ctx->stream));
    return YL_OK;
  }
  YL_CHECK(x && dy, YL_ERR_INVALID, "yl_layernorm_bwd: NULL argument");
  YL_CHECK(ldx >= cols && lddy >= cols && (!addend || ldadd >= cols) && (!dx || lddx >= cols),
           YL_ERR_SHAPE, "yl_layernorm_bwd: a row stride is smaller than %d columns", cols);
  const Span spans[] = {{dx, lddx, rows, cols}, {dgamma, cols, 1, cols},   {dbeta, cols, 1, cols},
                        {x, ldx, rows, cols},   {dy, lddy, rows, cols},    {addend, ldadd, rows, cols},
                        {gamma, cols, 1, cols}, {mean, rows, 1, rows},     {rstd, rows, 1, rows}};
  YL_CHECK(!results_overlap(spans, 3, 9, 0, 5), YL_ERR_INVALID,
           "yl_layernorm_bwd: a result overlaps another argument");
  if (!dx && !dgamma && !dbeta) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  Bwd p{x, dy, ldx, lddy, rows, cols, eps, gamma, mean, rstd, dx ? addend : nullptr, ldadd, dx, lddx,
        nullptr, nullptr, nullptr};
  const bool vec = aligned16(x) && aligned16(dy) && aligned16(gamma) && aligned16(p.addend) &&
                   aligned16(dx) && aligned16(dgamma) && aligned16(dbeta) &&
                   ((ldx | lddy | cols | (p.addend ? ldadd : 0) | (dx ? lddx : 0)) & 3) == 0;
  auto launch = [&](auto kernel, int threads, int rows_a_block, int unr, int smem) -> yl_status {
    long long blocks = (rows + rows_a_block - 1) / rows_a_block;
    // a few turns of one block are quicker than a second kernel for the sums
    if (blocks <= kAloneTurns && cols <= 16384) blocks = 1;
    YL_TRY(resident(ctx, kernel, threads, smem, &blocks));
    Workspace work;
    // rows a thread adds up per turn, turns per partial row, partial rows of a block
    const long long turns = (rows + blocks * rows_a_block - 1) / (blocks * rows_a_block);
    const long long per_part = kSegRows / unr;
    const long long parts = blocks * ((turns + per_part - 1) / per_part);
    if (parts == 1 && cols <= 16384) {
      p.dgamma = dgamma;
      p.dbeta = dbeta;
    } else if (dgamma || dbeta) {
      char* ws = nullptr;
      YL_TRY(work.get(ctx, (size_t)parts * 2 * cols * sizeof(float), &ws));
      p.part = (float*)ws;
    }
    kernel<<<(unsigned)blocks, threads, smem, ctx->stream>>>(p);
    YL_TRY(check_launch("ln_bwd_kernel"));
    if (p.part) {
      ln_bwd_columns_kernel<<<dim3((cols + 31) / 32, 2), 1024, 0, ctx->stream>>>(p.part, parts, cols,
                                                                                dgamma, dbeta);
      YL_TRY(check_launch("ln_bwd_columns_kernel"));
    }
    return work.done();
  };
  return vec ? bwd_aligned(cols, launch) : bwd_plain(cols, launch);
}

}  // extern "C"
