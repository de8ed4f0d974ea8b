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
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
#include <vector>

#include "yl_internal.h"
#include "yl_muon.h"
#include "yl_ptx.cuh"
#include "yl_ring.h"
#include "yume_c.h"

namespace yl {
namespace {

constexpr int kMaxSteps = 32;
// Largest singular value the iteration may reach on the way.
constexpr double kMaxSigma = 4.0;
constexpr int kMaxItems = 64;      // matrices of one launch's table
constexpr int kNormChunk = 4096;   // elements of one partial of a Frobenius norm
constexpr int kNormParts = 1024;   // most partials of one matrix: larger ones take longer chunks

// ---------------------------------------------------------------- data layout
// X, A and P live in the workspace as fp16 pairs: value * scale = hi + lo with
// hi the value rounded to fp16 and lo the rest rounded to fp16, 22 bits in all.
// A product of two pairs is hi hi + hi lo + lo hi, accumulated in fp32 on the
// tensor cores: as exact as an fp32 product (the dropped lo lo term is 2^-22 of
// a product), at a third of the fp16 rate, where the tf32 rate is half of it
// with 11 bits.  The scales are powers of two, per step, that keep the largest
// value the iteration can reach under fp16's range.  A pair has 22 bits down to
// 2^-17 of that value and none below 2^-40 of it, where an fp32 number goes on: so
// the scales of a matrix whose norm is far below eps start higher (below_one), and
// steps that would let what lies under that floor grow into the result are refused
// (plan_steps).
//
// Each plane (hi, lo) is a grid of 64 x 64 blocks of 8 KB whose bytes are
// already in the 128-byte-swizzled order the tensor core reads: 64 rows of 128
// bytes, 16-byte chunk j of row r at position j ^ (r & 7).  A block loads with
// one untiled bulk copy, needs no tensor map, and serves as a K-major or an
// MN-major operand alike, so tall matrices (X^T X on the left, X P) run from the
// same row-major blocks as wide ones (X X^T, P X) and nothing is transposed.
// Rows and columns past a matrix's edge are zeros inside its blocks.
constexpr int kBlk = 64;
constexpr int kBlkBytes = kBlk * kBlk * 2;

struct Item {
  const float* src;  // NS: x; Muon: the gradient
  float* mom;        // Muon: momentum, contiguous
  float* dst;        // NS: y; Muon: the parameter
  long long lds, ldd;
  int rows, cols;
  float scale;
  int rb, cb, mb;       // blocks of the rows, the columns and the shorter side
  uint8_t *x[2], *a, *p;  // workspace: pairs of planes (X before and after a step, A, P)
  double* part;         // partial sums of squares
  int chunks;
  int chunk;            // elements of one partial
  int vec;              // 16-byte loads of src and mom: 1 everywhere
  int narrow;           // bit of a phase: its tiles have 64 columns, not 128
  int ks;               // GRAM: shares of the long side, each a ticket of its own
  int split0;           // its first arrival counter
  float* partial;       // [GRAM tile][share][column][row] sums of the shares
};
enum { GRAM = 0, SQUARE = 1, UPDATE = 2 };
constexpr int kPairSide = 512;
constexpr int kMaxShares = 64;
struct Table {
  Item it[kMaxItems];
  int tiles[3][kMaxItems + 1];  // GRAM, SQUARE, UPDATE tickets before each item
  int blocks[kMaxItems + 1];    // 64 x 64 blocks of X before each item
  int chunks[kMaxItems + 1];    // norm chunks before each item
  int count;
  int pair;                     // worked on by pairs of blocks, 256 x 256 tiles
  int chip;                     // stays in shared memory
  int below[kMaxItems];         // below_one of each item, from the split pass
  int* ctrl;                    // ticket counter, done[item][3], arrivals of split GRAM tiles
  int ctrl_ints;
};
constexpr int kCtrlDone = 1, kCtrlSplit = kCtrlDone + 3 * kMaxItems;
struct Update {
  int muon, nesterov, sanitize;
  float mu, lr, decay, grad_scale, clip, eps;
  const float* norm;
};

__device__ __forceinline__ int find_item(const int* start, int count, int t) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
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
// What is orthogonalised: x itself, or the momentum (with Nesterov's look ahead).
__device__ __forceinline__ float update_value(const Item& it, const Update& u, float clipf,
                                              long long r, long long c) {
  if (!u.muon) return it.src[r * it.lds + c];
  const long long i = r * it.cols + c;
  const float m = it.mom[i];
  return u.nesterov ? clean(it.src[i], u, clipf) + u.mu * m : m;
}

// Sum over a block of 256 threads in a fixed order, the same in every thread.
__device__ __forceinline__ double block_sum256(double s) {
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  double t = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += red[w];
  return t;
}

// The momentum step and the partial sums of squares of u; block 0 also leaves
// the table in device memory for the kernels that follow.
__global__ void __launch_bounds__(256)
    ns_norm_kernel(const __grid_constant__ Table t, const __grid_constant__ Update u,
                   Table* table_out) {
  if (blockIdx.x == 0) {
    const int* s = reinterpret_cast<const int*>(&t);
    int* d = reinterpret_cast<int*>(table_out);
    for (int i = threadIdx.x; i < (int)(sizeof(Table) / 4); i += 256) d[i] = s[i];
    for (int i = threadIdx.x; i < t.ctrl_ints; i += 256) t.ctrl[i] = 0;
  }
  const int k = find_item(t.chunks, t.count, blockIdx.x);
  const Item& it = t.it[k];
  const int chunk = blockIdx.x - t.chunks[k];
  const long long total = (long long)it.rows * it.cols;
  const long long lo = (long long)chunk * it.chunk;
  const int n = (int)min((long long)it.chunk, total - lo);
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  double s = 0.0;
  if (u.muon) {
    const float* g = it.src + lo;
    float* mo = it.mom + lo;
    auto one = [&](float graw, float& m) {
      const float gv = clean(graw, u, clipf);
      m = u.mu * m + gv;
      const float v = u.nesterov ? gv + u.mu * m : m;
      s += (double)v * v;
    };
    int i = 0;
    if (it.vec) {
#pragma unroll 2
      for (i = threadIdx.x; i < n / 4; i += 256) {
        const float4 gv = __ldg(reinterpret_cast<const float4*>(g) + i);
        float4 m = reinterpret_cast<const float4*>(mo)[i];
        one(gv.x, m.x), one(gv.y, m.y), one(gv.z, m.z), one(gv.w, m.w);
        reinterpret_cast<float4*>(mo)[i] = m;
      }
      i = n & ~3;
    }
#pragma unroll 4
    for (i += threadIdx.x; i < n; i += 256) {
      float m = mo[i];
      one(__ldg(g + i), m);
      mo[i] = m;
    }
  } else if (it.lds == it.cols) {
    const float* x = it.src + lo;
    auto one = [&](float v) { s += (double)v * v; };
    int i = 0;
    if (it.vec) {
#pragma unroll 4
      for (i = threadIdx.x; i < n / 4; i += 256) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(x) + i);
        one(v.x), one(v.y), one(v.z), one(v.w);
      }
      i = n & ~3;
    }
#pragma unroll 4
    for (i += threadIdx.x; i < n; i += 256) one(__ldg(x + i));
  } else {  // strided rows: walk (row, column) without a division per element
    const long long i0 = lo + threadIdx.x;
    long long r = i0 / it.cols;
    int c = (int)(i0 - r * it.cols);
    const int dr = 256 / it.cols, dc = 256 - dr * it.cols;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) {
      const float v = __ldg(it.src + r * it.lds + c);
      s += (double)v * v;
      r += dr;
      c += dc;
      if (c >= it.cols) c -= it.cols, ++r;
    }
  }
  s = block_sum256(s);
  if (threadIdx.x == 0) it.part[chunk] = s;
}

// part[block] = sum of squares of one chunk of scaled (and sanitized) gradients
__global__ void __launch_bounds__(256)
    grad_square_kernel(const float* __restrict__ g, long long n, float scale, int sanitize,
                       double* __restrict__ part) {
  const long long lo = blockIdx.x * (long long)kNormChunk;
  const long long hi = min(n, lo + (long long)kNormChunk);
  double s = 0.0;
  for (long long i = lo + threadIdx.x; i < hi; i += 256) {
    float v = g[i] * scale;
    if (sanitize && !isfinite(v)) v = 0.f;
    s += (double)v * v;
  }
  s = block_sum256(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}
// The same over a table's gradients.
__global__ void __launch_bounds__(256)
    table_square_kernel(const __grid_constant__ Table t, float scale, int sanitize,
                        double* __restrict__ part) {
  const int k = find_item(t.chunks, t.count, blockIdx.x);
  const Item& it = t.it[k];
  const long long lo = (long long)(blockIdx.x - t.chunks[k]) * it.chunk;
  const int n = (int)min((long long)it.chunk, (long long)it.rows * it.cols - lo);
  const float* g = it.src + lo;
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) {
    float v = __ldg(g + i) * scale;
    if (sanitize && !isfinite(v)) v = 0.f;
    s += (double)v * v;
  }
  s = block_sum256(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}
__global__ void __launch_bounds__(256)
    grad_norm_final_kernel(const double* __restrict__ part, long long n, float* norm) {
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += 256) s += part[i];
  s = block_sum256(s);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// 1 / (sqrt(sum of squares) + eps); 0 for a zero matrix, NaN for one with a NaN or
// an infinity.  In double, for matrices whose norm's inverse is no float.
__device__ __forceinline__ double inverse_norm(double squares, float eps) {
  if (squares == 0.0) return 0.0;
  const double norm = sqrt(squares);
  return isinf(norm) ? __longlong_as_double(0x7ff8000000000000LL) : 1.0 / (norm + (double)eps);
}
__device__ __forceinline__ double item_squares(const Item& it) {
  double s = 0.0;
  for (int c = threadIdx.x; c < it.chunks; c += 256) s += it.part[c];
  return block_sum256(s);
}
// X0's norm |u| / (|u| + eps) is at most 2^-(what this returns): 0 unless eps is the
// larger of the two.
constexpr int kMaxBelow = 120;  // X0's values are then at the end of fp32's range
__device__ __forceinline__ int below_one(double squares, float eps) {
  const double norm = sqrt(squares), e = (double)eps;
  if (!(norm > 0.0 && norm < e)) return 0;
  const double ratio = norm / (norm + e);
  return ratio > 0.0 ? max(0, min(kMaxBelow, -1 - ilogb(ratio))) : 0;
}

__device__ __forceinline__ void split_pair(float v, __half* hi, __half* lo) {
  *hi = __float2half_rn(v);
  *lo = __float2half_rn(v - __half2float(*hi));
}

// X0 = u / (|u| + eps) as fp16 pairs, one 64 x 64 block per thread block; each
// thread fills two 16-byte chunks of either plane.
__global__ void __launch_bounds__(256)
    ns_split_kernel(const Table* __restrict__ t, const __grid_constant__ Update u, float sx,
                    int* __restrict__ below_out) {
  // from the end, which the pass before has left in L2 (39 of the U-Net's weights 442 us,
  // from the start 445)
  const int at0 = gridDim.x - 1 - blockIdx.x, k = find_item(t->blocks, t->count, at0);
  const Item& it = t->it[k];
  const int b = at0 - t->blocks[k];
  const int rb = b / it.cb, cb = b - rb * it.cb;
  const double squares = item_squares(it);
  const int below = below_one(squares, u.eps);
  double inv = inverse_norm(squares, u.eps);
  if (below) inv = ldexp(inv, below);
  if (b == 0 && threadIdx.x == 0) below_out[k] = below;
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  uint8_t* hi = it.x[0] + (size_t)b * kBlkBytes;
  uint8_t* lo = hi + (size_t)it.rb * it.cb * kBlkBytes;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int idx = threadIdx.x + 256 * e, row = idx >> 3, ch = idx & 7;
    const long long r = (long long)rb * kBlk + row, c0 = (long long)cb * kBlk + ch * 8;
    float v[8];
    if (it.vec && r < it.rows && c0 + 8 <= it.cols) {
      const float* x = it.src + r * it.lds + c0;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float4 g = make_float4(0.f, 0.f, 0.f, 0.f), m = g;
        if (!u.muon || u.nesterov) g = __ldg(reinterpret_cast<const float4*>(x) + q);
        if (u.muon) m = __ldg(reinterpret_cast<const float4*>(it.mom + r * it.cols + c0) + q);
        const float ge[4] = {g.x, g.y, g.z, g.w}, me[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[4 * q + j] = !u.muon ? ge[j]
                         : u.nesterov ? clean(ge[j], u, clipf) + u.mu * me[j]
                                      : me[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = r < it.rows && c0 + j < it.cols ? update_value(it, u, clipf, r, c0 + j) : 0.f;
    }
    __align__(16) __half h[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) split_pair((float)(v[j] * inv) * sx, &h[j], &l[j]);
    const int at = row * 128 + ((ch ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(hi + at) = *reinterpret_cast<const uint4*>(h);
    *reinterpret_cast<uint4*>(lo + at) = *reinterpret_cast<const uint4*>(l);
  }
}

// No step at all: y = X0 (or the update with it).
__global__ void __launch_bounds__(256)
    ns_direct_kernel(const Table* __restrict__ t, const __grid_constant__ Update u) {
  const int k = find_item(t->chunks, t->count, blockIdx.x);
  const Item& it = t->it[k];
  const int chunk = blockIdx.x - t->chunks[k];
  const double inv = inverse_norm(item_squares(it), u.eps);
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  const long long total = (long long)it.rows * it.cols;
  const long long lo = (long long)chunk * it.chunk;
  const long long hi = min(total, lo + (long long)it.chunk);
  for (long long i = lo + threadIdx.x; i < hi; i += 256) {
    const long long r = i / it.cols, c = i - r * it.cols;
    const float v = (float)(update_value(it, u, clipf, r, c) * inv);
    if (u.muon) it.dst[i] = it.dst[i] * (1.f - u.lr * u.decay) - u.lr * it.scale * v;
    else it.dst[r * it.ldd + c] = v;
  }
}

// ---------------------------------------------------------------- products
// All steps of all matrices in one persistent kernel.  Its work is a list of
// tickets, 128 x 128 tiles of
//   GRAM    A = X X^T (X^T X for tall matrices), tiles on and below the diagonal;
//           the long side may be split into shares whose sums the last one to
//           finish adds up in share order;
//   SQUARE  P = a I + b A + c A A, tiles on and below the diagonal;
//   UPDATE  X' = P X (X P), or in the last step the result itself,
// step by step, phase by phase, matrix by matrix.  A thread block takes the next
// ticket from a counter; before it loads a tile it waits until that matrix's
// tiles of the phase before are done.  Tickets are handed out in an order in
// which every tile comes after the tiles it needs, and a taken ticket belongs to
// a running block, so the waits end however many blocks are resident.
//
// Warp 10 takes the tickets and works out what they are, which with its trips to
// memory takes 2.3 us (behind warp 8's loads it held up every tile: 2048 x 2048
// 576 us, with a warp of its own 526).  Warp 8 streams operand blocks (128 x 64 of
// either side, both planes: 64 KB a stage; half of that on the diagonal, where both
// sides are the same) through a ring of three stages, warp 9 issues the
// tcgen05.mma, and warps 0-7 add each finished accumulator into registers (64
// columns of 32 rows per warp) and write the tile.
// The tensor core truncates when it adds to its accumulator: kept there over a
// whole row, a 384 x 1153 matrix ended 2.4e-5 off, where an fp32 product gives
// 2e-6.  So an accumulator takes a few 16-deep products only, the small ones
// (hi lo, lo hi) of a k-block first, and the sum over the row is in registers with
// fp32's rounding.  What costs accuracy is a term far above the others, and A and
// P have theirs on the diagonal: with two k-blocks to an accumulator throughout
// 256 x 2304 ended 7.3e-6 off, with two in GRAM and half a k-block elsewhere 2.1e-6
// (fp32: 2.0e-6).  So it is one k-block where the tile meets the diagonal, two
// elsewhere, whose handover then hides behind the tensor core's work.
// What truncation takes off depends on the data: about 2^-22 of a product of dense
// operands (eight additions to an accumulator, half a last place of half the sum each),
// nothing where a sum has one term.  scaled_steps puts half of the former back in GRAM
// and SQUARE, so that neither kind of matrix has the whole of it left.  Mean errors
// over eight seeds against those of fp32 products, normal and diagonal matrices, the
// worst of seven shapes each: on the chip 1.4 and 1.4 (nothing put back 2.0 and 1.9,
// all of it, 2^-22 in both and 2^-23 in UPDATE, 1.4 and 3.0), in tiles with a shorter
// side past 128 1.1 and 1.5 (1.3 and 1.5; 0.8 and 3.9), with a shorter one 2.7, at 64 x
// 1000, and 1.6 (3.3 and 1.5; 1.6 and 3.7).
//
// Two forms.  A single block works on 128 x 128 tiles; its MMAs are bound by their
// reads of shared memory (12 of 128 x 128 a k-block, 8 KB each, take 117 cycles
// each, not 64), so the left hi plane meets both right planes in one of 256 columns
// (12 KB).  With the copies' writes (64 KB) that is 144 KB of a k-block through shared
// memory, at 128 bytes a cycle its 1.1k cycles.  Tiles of 64 columns (`narrow`) move
// 104 KB and take 0.8k: more per product, but twice the tiles, each sooner done,
// where SMs are idle.  A pair
// of blocks (PAIR: a cluster of two, cta_group::2) works on 256 x 256 tiles, each
// block with half of the rows of both sides: the same 8 KB of reads for four
// times the products, 128 cycles per block, bound by the tensor cores.
constexpr int kStages = 3;
constexpr int kOpBytes = 2 * kBlkBytes;       // one plane of one block's 128 rows x 64
constexpr int kStageBytes = 4 * kOpBytes;     // L hi, L lo, R hi, R lo
constexpr int kOutOff = kStages * kStageBytes;
constexpr int kOutWarp = 4096;                // staging of one epilogue warp
constexpr int kEpiWarps = 8;
constexpr int kBarOff = kOutOff + kEpiWarps * kOutWarp;
constexpr int kSmemBytes = kBarOff + 1536 + 1024;  // barriers and prefixes, alignment
// Three warpgroups of 168 registers a thread at launch; the two of the epilogue
// take over what the third does not need: 2 * 216 + 72 = 3 * 168.
constexpr int kProductThreads = 384;
constexpr int kRegsEpilogue = 216, kRegsOthers = 72;
constexpr int kRing = 4;     // tickets on their way from the scheduler to the other warps
// k-blocks left to load when the next ticket is taken: 1 costs as much on large
// tables and 1% more on those of many short tickets
constexpr int kAskAhead = 4;
constexpr int kTmemCols = 512;

template <bool PAIR>
struct Form {
  static constexpr int kCtas = PAIR ? 2 : 1;
  static constexpr int kTile = 128 * kCtas;            // rows and columns of a tile
  static constexpr int kSide = 2 * kCtas;              // blocks along it
  static constexpr int kAccCols = 256;                 // one accumulator in TMEM
  static constexpr int kAccs = kTmemCols / kAccCols;
  static constexpr int kCols = kTile / 2;              // columns of one epilogue warp
};

struct Steps {
  int n;
  float g2[kMaxSteps];                                // GRAM: A' = g2 acc
  float s0[kMaxSteps], s1[kMaxSteps], s2[kMaxSteps];  // SQUARE: P' = s0 I + s1 A' + s2 acc
  float u2[kMaxSteps];                                // UPDATE: X' = u2 acc
  // X grows by at most 2^rise[k] before step k, against the bounds of the scales
  int rise[kMaxSteps + 1];
};

// The factors of a matrix that starts `below` powers of two under the scales' bound:
// X is kept by 2^s larger and A by 2^(2 s), as long as that still counts in P (A less
// than 2^-60 of the identity's part does not), until the growth of the steps has
// used it up.
struct Lift {
  int s, a;
  __device__ Lift(const Steps& st, int below, int step)
      : s(max(0, below - st.rise[step])), a(min(2 * s, 60)) {}
  __device__ float gram(float g2) const { return ldexpf(g2, a - 2 * s); }
  __device__ float linear(float s1) const { return ldexpf(s1, -a); }
  __device__ float square(float s2) const { return ldexpf(s2, -2 * a); }
  // (the last step's result is not kept at a scale)
  __device__ float update(const Steps& st, int below, int step, float u2) const {
    return ldexpf(u2, (step + 1 == st.n ? 0 : max(0, below - st.rise[step + 1])) - s);
  }
};

struct Ticket {
  int step, mode, item, i, j, kb0, nk, share, tile;
  float c2, s1;  // the tile is c2 times its sums (+ s1 A + s0 I)
};
constexpr int kTicketInts = sizeof(Ticket) / 4, kNoTicket = -1;  // mode behind the last one

// `start` is the table's tiles[3][kMaxItems + 1] in shared memory.
template <bool PAIR, bool NARROW>
__device__ __forceinline__ Ticket ticket_of(const Table* t, const int* start, int count, int n) {
  Ticket q;
  const int gram = start[count], square = start[kMaxItems + 1 + count];
  const int per = gram + square + start[2 * (kMaxItems + 1) + count];
  q.step = n / per;
  n -= q.step * per;
  q.mode = GRAM;
  if (n >= gram) {
    n -= gram;
    q.mode = SQUARE;
    if (n >= square) {
      n -= square;
      q.mode = UPDATE;
    }
  }
  const int* st = start + q.mode * (kMaxItems + 1);
  q.item = find_item(st, count, n);
  const Item& it = t->it[q.item];
  int k = n - st[q.item];
  q.kb0 = 0;
  q.share = 0;
  q.nk = it.mb;
  const bool narrow = NARROW && (it.narrow >> q.mode & 1);
  if (q.mode == UPDATE) {
    const int tn = narrow ? it.cb : (it.cb + Form<PAIR>::kSide - 1) / Form<PAIR>::kSide;
    q.i = k / tn;
    q.j = k - q.i * tn;
    q.tile = k;
    return q;
  }
  if (q.mode == GRAM) {
    const int nk = it.rows > it.cols ? it.rb : it.cb, ks = it.ks;
    q.share = k % ks;
    k /= ks;
    q.kb0 = (int)((long long)nk * q.share / ks);
    q.nk = (int)((long long)nk * (q.share + 1) / ks) - q.kb0;
  }
  q.tile = k;
  if (narrow) {  // lower triangle, row by row, 2 i + 2 tiles in row i: k = i (i + 1) + j
    int i = (int)((sqrtf(4.f * k + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) > k) --i;
    while ((i + 1) * (i + 2) <= k) ++i;
    q.i = i;
    q.j = k - i * (i + 1);
    return q;
  }
  // lower triangle, row by row: k = i (i + 1) / 2 + j
  int i = (int)((sqrtf(8.f * k + 1.f) - 1.f) * 0.5f);
  while (i * (i + 1) / 2 > k) --i;
  while ((i + 1) * (i + 2) / 2 <= k) ++i;
  q.i = i;
  q.j = k - i * (i + 1) / 2;
  return q;
}

// The row of tiles that a ticket's columns are.
template <bool NARROW>
__device__ __forceinline__ int column_tile(const Item& it, const Ticket& q) {
  return NARROW && (it.narrow >> q.mode & 1) ? q.j >> 1 : q.j;
}

// Whether k-block kb of a ticket meets the diagonal of A or P.
template <bool PAIR, bool NARROW>
__device__ __forceinline__ bool on_diagonal(const Item& it, const Ticket& q, int kb) {
  const int kt = kb / Form<PAIR>::kSide;
  if (q.mode == GRAM) return false;
  const int jt = column_tile<NARROW>(it, q);
  if (q.mode == SQUARE) return kt == q.i || kt == jt;
  return kt == (it.rows > it.cols ? jt : q.i);
}

// One operand: block (mn, k) of a plane is at base + (mn * smn + k * sk) blocks.
// Of A and P (sym) only the tiles on and below the diagonal are kept: a block
// above it is read from its mirror image, as an MN-major operand.
struct Operand {
  const uint8_t* base;
  size_t plane;  // bytes from the hi to the lo plane
  int smn, sk, nmn;
  int mn_major;
  int sym;
};
__device__ __forceinline__ Operand operand(const Item& it, int mode, int from, int right) {
  const bool tall = it.rows > it.cols;
  const uint8_t* x = it.x[from];
  const size_t xp = (size_t)it.rb * it.cb * kBlkBytes, mp = (size_t)it.mb * it.mb * kBlkBytes;
  if (mode == GRAM)  // rows of X, or columns when tall
    return {x, xp, tall ? 1 : it.cb, tall ? it.cb : 1, it.mb, tall, 0};
  if (mode == SQUARE) return {it.a, mp, it.mb, 1, it.mb, 0, 1};
  if (tall != (right != 0))  // X's rows (tall, left) or columns (wide, right)
    return {x, xp, right ? 1 : it.cb, right ? it.cb : 1, right ? it.cb : it.rb, right, 0};
  return {it.p, mp, it.mb, 1, it.mb, 0, 1};
}

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void add_release(int* p, int v) {
  asm volatile("fence.acq_rel.gpu; red.relaxed.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// (the fence for every state space costs 0.35 us more, in front of every tile)
__device__ __forceinline__ void fence_proxy_async_global() {
  asm volatile("fence.proxy.async.global;" ::: "memory");
}

// The counter a ticket waits for, and the value it must have reached (every
// block of a tile counts).
template <bool PAIR>
__device__ __forceinline__ const int* needs(const Table* t, const int* start, const Ticket& q,
                                            int* value) {
  const int before = (q.mode + 2) % 3;  // GRAM <- UPDATE of the step before
  const int* st = start + before * (kMaxItems + 1) + q.item;
  int tiles = st[1] - st[0];
  if (before == GRAM) tiles /= t->it[q.item].ks;  // counted once per tile
  *value = Form<PAIR>::kCtas * tiles * (q.mode == GRAM ? q.step : q.step + 1);
  return t->ctrl + kCtrlDone + 3 * q.item + before;
}

template <bool PAIR>
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, long long lim) {
  return PAIR ? mbar_wait_cluster(bar, parity, lim) : mbar_wait(bar, parity, lim);
}

// NARROW: some of the table's matrices are.
template <bool PAIR, bool NARROW>
__global__ void __launch_bounds__(kProductThreads, 1)
    ns_steps_kernel(const Table* __restrict__ t, const __grid_constant__ Steps steps,
                    const __grid_constant__ Update u, int* err) {
  using F = Form<PAIR>;
  constexpr int kAccs = F::kAccs, kCols = F::kCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBarOff);  // this block's copies
  uint64_t* pfull = full + kStages;       // rank 0: the other block's copies
  uint64_t* empty = pfull + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + kAccs;  // rank 0
  uint64_t* tfull = acc_empty + kAccs;
  uint64_t* tempty = tfull + kRing;        // rank 0
  uint64_t* ready = tempty + kRing;        // the ticket's operands are there
  uint64_t* ask = ready + kRing;           // rank 0
  uint64_t* drain = ask + 1;
  uint64_t* esync = drain + 1;
  uint64_t* seen = esync + 1;              // [2]: a SQUARE tile's own A may be freed
  Ticket* ring = reinterpret_cast<Ticket*>(seen + 2);
  int* last_share = reinterpret_cast<int*>(ring + kRing);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last_share + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 1);  // [3][kMaxItems + 1]
  int* below = start + 3 * (kMaxItems + 1);            // [kMaxItems]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int count = t->count;
  for (int i = threadIdx.x; i < 3 * (kMaxItems + 1); i += kProductThreads)
    start[i] = (&t->tiles[0][0])[i];
  for (int i = threadIdx.x; i < count; i += kProductThreads) below[i] = t->below[i];
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&pfull[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kAccs; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], F::kCtas * kEpiWarps);
    }
    for (int b = 0; b < kRing; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&ready[b], 1);
      // rank 0: producer, MMA thread, epilogue; rank 1: these (as relay) and the scheduler
      mbar_init(&tempty[b], 2 + kEpiWarps + (PAIR ? 3 + kEpiWarps : 0));
    }
    mbar_init(ask, 1);
    mbar_init(drain, 1);
    mbar_init(esync, kEpiWarps);
    for (int b = 0; b < 2; ++b) mbar_init(&seen[b], 1);
    fence_barrier_init();
  }
  if (PAIR) {
    __syncthreads();
    cluster_sync_all();  // the other block's barriers are ready, and both can allocate
  }
  if (warp == kEpiWarps + 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, kTmemCols);
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = steps.n * (start[count] + start[kMaxItems + 1 + count] +
                               start[2 * (kMaxItems + 1) + count]);
  const long long lim = wait_limit(err);
  // arrivals on rank 0's barriers
  auto arrive0 = [&](uint64_t* bar) {
    if (PAIR) mbar_arrive_cluster(map_to_rank(smem_u32(bar), 0));
    else mbar_arrive(bar);
  };

  if (warp >= kEpiWarps) {
    reg_dec<kRegsOthers>();
  if (warp == kEpiWarps + 2) {
    // scheduler: takes the tickets and waits until what they need is done
    if (lane == 0) {
      for (uint32_t k = 0;; ++k) {
        const int slot = k % kRing;
        Ticket q;
        if (rank == 0) {
          // taken no earlier than its loads could nearly start: a ticket held back
          // here is one that an idle block would have begun
          if ((k > 0 && !mbar_wait(ask, (k - 1) & 1, lim)) ||
              (k >= kRing && !wait<PAIR>(&tempty[slot], (k / kRing - 1) & 1, lim))) {
            report_error(err, YL_DEVERR_TIMEOUT);
            break;
          }
          const int n = atomicAdd(t->ctrl, 1);
          q.mode = kNoTicket;
          if (n < total) {
            q = ticket_of<PAIR, NARROW>(t, start, count, n);
            // (looked up here and not in the epilogue, which every tile waits for: 512 x 512
            // and 512 x 128 148.4 us, there 150.8)
            q.c2 = q.mode == GRAM     ? steps.g2[q.step]
                   : q.mode == SQUARE ? steps.s2[q.step]
                                      : steps.u2[q.step];
            q.s1 = steps.s1[q.step];
            if (const int e = below[q.item]) {
              const Lift lift(steps, e, q.step);
              q.c2 = q.mode == GRAM     ? lift.gram(q.c2)
                     : q.mode == SQUARE ? lift.square(q.c2)
                                        : lift.update(steps, e, q.step, q.c2);
              q.s1 = lift.linear(q.s1);
            }
          }
          ring[slot] = q;
          mbar_arrive(&tfull[slot]);
          if (PAIR) {
            const int* words = reinterpret_cast<const int*>(&ring[slot]);
            const uint32_t there = map_to_rank(smem_u32(words), 1);
#pragma unroll
            for (int w = 0; w < kTicketInts; ++w) st_cluster_s32(there + 4 * w, words[w]);
            mbar_arrive_cluster(map_to_rank(smem_u32(&tfull[slot]), 1));
          }
        } else {
          if (!wait<PAIR>(&tfull[slot], (k / kRing) & 1, lim)) {
            report_error(err, YL_DEVERR_TIMEOUT);
            break;
          }
          q = ring[slot];
          arrive0(&tempty[slot]);
        }
        if (q.mode == kNoTicket) break;
        int value;
        const int* counter = needs<PAIR>(t, start, q, &value);
        const long long t0 = clock64();
        bool ok = true;
        while (ok && load_acquire(counter) < value) ok = clock64() - t0 <= lim;
        if (!ok) {
          report_error(err, YL_DEVERR_TIMEOUT);
          break;
        }
        mbar_arrive(&ready[slot]);
      }
    }
  } else if (warp == kEpiWarps) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t k = 0; ok; ++k) {
        const int slot = k % kRing;
        if (!wait<PAIR>(&tfull[slot], (k / kRing) & 1, lim)) {
          report_error(err, YL_DEVERR_TIMEOUT);
          break;
        }
        const Ticket q = ring[slot];
        arrive0(&tempty[slot]);
        if (q.mode == kNoTicket) break;
        const Item& im = t->it[q.item];
        const Operand L = operand(im, q.mode, q.step & 1, 0), R = operand(im, q.mode, q.step & 1, 1);
        const bool narrow = NARROW && (im.narrow >> q.mode & 1);
        const bool same = !narrow && q.mode != UPDATE && q.i == q.j;
        const int l0 = F::kSide * q.i + 2 * rank, r0 = narrow ? q.j : F::kSide * q.j + 2 * rank;
        const int nl = max(0, min(2, L.nmn - l0));
        const int nr = same ? 0 : max(0, min(narrow ? 1 : 2, R.nmn - r0));
        const int jt = column_tile<NARROW>(im, q);
        if (!mbar_wait(&ready[slot], (k / kRing) & 1, lim)) {
          report_error(err, YL_DEVERR_TIMEOUT);
          break;
        }
        const int extra = q.mode == SQUARE ? F::kCtas : 0;  // stages with the tile's own A
        fence_proxy_async_global();  // what the scheduler saw, before this thread's bulk loads
        const int ask_at = max(0, q.nk + extra - kAskAhead);
        for (int kb = 0; kb < q.nk + extra; ++kb, ++it) {
          if (kb == ask_at && rank == 0) mbar_arrive(ask);
          const int s = it % kStages;
          if (it >= kStages && !wait<PAIR>(&empty[s], ((it / kStages) - 1) & 1, lim)) {
            report_error(err, YL_DEVERR_TIMEOUT);
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(smem + s * kStageBytes);
          if (kb >= q.nk) {  // 128 rows x 128 columns of A for the epilogue, blocks [row][column]
            const int c0 = narrow ? q.j : F::kSide * q.j + 2 * (kb - q.nk);
            const int nc = max(0, min(narrow ? 1 : 2, im.mb - c0));
            mbar_arrive_expect_tx(&full[s], (uint32_t)(2 * nl * nc) * kBlkBytes);
            for (int b = 0; b < nl * nc; ++b) {
              const int br = b / nc, bc = b - br * nc;
              const uint8_t* src = im.a + ((size_t)(l0 + br) * im.mb + c0 + bc) * kBlkBytes;
              const uint32_t d = dst + (uint32_t)((2 * br + bc) * kBlkBytes);
              bulk_load(d, src, kBlkBytes, &full[s]);
              bulk_load(d + 2 * kOpBytes, src + L.plane, kBlkBytes, &full[s]);
            }
            continue;
          }
          mbar_arrive_expect_tx(&full[s], (uint32_t)(2 * (nl + nr)) * kBlkBytes);
          const int kk = q.kb0 + kb;
          for (int side = 0; side < 2; ++side) {
            const Operand& o = side ? R : L;
            const int nb = side ? nr : nl, mn0 = side ? r0 : l0;
            const bool above = o.sym && (side ? jt : q.i) < kk / F::kSide;
            const uint32_t lo = side && narrow ? kBlkBytes : kOpBytes;  // its lo plane
            const size_t smn = above ? o.sk : o.smn, sk = above ? o.smn : o.sk;
            for (int b = 0; b < nb; ++b) {
              const uint8_t* src = o.base + ((size_t)(mn0 + b) * smn + (size_t)kk * sk) * kBlkBytes;
              const uint32_t d = dst + (uint32_t)(side * 2 * kOpBytes + b * kBlkBytes);
              bulk_load(d, src, kBlkBytes, &full[s]);
              bulk_load(d + lo, src + o.plane, kBlkBytes, &full[s]);
            }
          }
        }
      }
      drain_ring(full, kStages, it);  // no copy may still be landing when the block exits
    }
  } else if (warp == kEpiWarps + 1) {
    if (lane == 0) {
      uint32_t it = 0, ci = 0, squares = 0;
      bool ok = true;
      auto commit = [&](uint64_t* bar) {
        if (PAIR) umma_commit_pair(bar);
        else umma_commit(bar);
      };
      for (uint32_t k = 0; ok; ++k) {
        const int slot = k % kRing;
        if (!wait<PAIR>(&tfull[slot], (k / kRing) & 1, lim)) {
          report_error(err, YL_DEVERR_TIMEOUT);
          break;
        }
        const Ticket q = ring[slot];
        arrive0(&tempty[slot]);
        if (q.mode == kNoTicket) break;
        const int extra = q.mode == SQUARE ? F::kCtas : 0;
        if (rank != 0) {  // tell rank 0 of every stage that has landed here
          for (int kb = 0; kb < q.nk + extra; ++kb, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(&full[s], (it / kStages) & 1, lim)) {
              report_error(err, YL_DEVERR_TIMEOUT);
              ok = false;
              break;
            }
            arrive0(&pfull[s]);
          }
          continue;
        }
        const Item& im = t->it[q.item];
        const Operand L = operand(im, q.mode, 0, 0), R = operand(im, q.mode, 0, 1);
        const bool narrow = NARROW && (im.narrow >> q.mode & 1);
        const bool same = !narrow && q.mode != UPDATE && q.i == q.j;
        const int jt = column_tile<NARROW>(im, q);
        int filled = 0;  // k-blocks the current accumulator has taken
        for (int kb = 0; ok && kb < q.nk; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&full[s], (it / kStages) & 1, lim) ||
              (PAIR && !wait<PAIR>(&pfull[s], (it / kStages) & 1, lim))) {
            report_error(err, YL_DEVERR_TIMEOUT);
            ok = false;
            break;
          }
          const int kt = (q.kb0 + kb) / F::kSide;
          const int lmn = L.mn_major | (L.sym & (q.i < kt)), rmn = R.mn_major | (R.sym & (jt < kt));
          const int cols = narrow ? 64 : F::kTile;
          const uint32_t idesc = idesc_f16(F::kTile, cols, lmn, rmn);
          // K-major: 16 of a row's 64 k are 32 bytes, 8-row groups 1 KB apart.
          // MN-major: 16 k are two 8-row groups, 64-column blocks 8 KB apart.
          const uint32_t lstep = lmn ? 2048 : 32, rstep = rmn ? 2048 : 32;
          const uint32_t llbo = lmn ? kBlkBytes : 16, rlbo = rmn ? kBlkBytes : 16;
          const uint32_t l = smem_u32(smem + s * kStageBytes), r = same ? l : l + 2 * kOpBytes;
          const bool fine = on_diagonal<PAIR, NARROW>(im, q, kb);
          const int buf = ci % kAccs;
          if (filled == 0 && ci >= kAccs && !wait<PAIR>(&acc_empty[buf], (ci / kAccs - 1) & 1, lim)) {
            report_error(err, YL_DEVERR_TIMEOUT);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t dacc = tmem + (uint32_t)(buf * F::kAccCols);
          if constexpr (PAIR) {
#pragma unroll
            for (int part = 0; part < 3; ++part) {  // lo hi, hi lo, hi hi
              const uint32_t lp = l + (part == 0 ? kOpBytes : 0);
              const uint32_t rp = r + (part == 1 ? kOpBytes : 0);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_f16_pair(dacc, sw128_desc(lp + kk * lstep, llbo, 1024),
                              sw128_desc(rp + kk * rstep, rlbo, 1024), idesc,
                              (filled | part | kk) != 0);
            }
          } else {
            // both planes of the right side lie one behind the other: hi (hi | lo) is
            // one product of twice the columns, lo hi goes to the second half of them
            const uint32_t wide = idesc_f16(128, 2 * cols, lmn, rmn);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16(dacc, sw128_desc(l + kk * lstep, llbo, 1024),
                       sw128_desc(r + kk * rstep, rlbo, 1024), wide, (filled | kk) != 0);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16(dacc + cols, sw128_desc(l + kOpBytes + kk * lstep, llbo, 1024),
                       sw128_desc(r + kk * rstep, rlbo, 1024), idesc, 1);
          }
          if (++filled == 2 || fine || kb + 1 == q.nk || on_diagonal<PAIR, NARROW>(im, q, kb + 1)) {
            commit(&acc_full[buf]);
            filled = 0;
            ++ci;
          }
          commit(&empty[s]);
        }
        if (!ok || extra == 0) continue;
        ok = pass_stages(it, extra, [&](uint32_t i) {
          return mbar_wait(&full[i % kStages], (i / kStages) & 1, lim) &&
                 (!PAIR || wait<PAIR>(&pfull[i % kStages], (i / kStages) & 1, lim));
        });
        if (!ok) {
          report_error(err, YL_DEVERR_TIMEOUT);
        } else {  // the epilogue may free what this thread has seen
          uint64_t* bar = &seen[squares++ & 1];
          mbar_arrive(bar);
          if (PAIR) mbar_arrive_cluster(map_to_rank(smem_u32(bar), 1));
        }
      }
      // every MMA this thread issued has completed before TMEM and the other
      // block's shared memory are released
      if (rank == 0) commit(drain);
      wait<PAIR>(drain, 0, kWaitLimitCycles);
    }
  }
  } else {
    reg_inc<kRegsEpilogue>();
    // epilogue: warp w owns rows 32 (w % 4) .. + 31 of the block's 128 (its TMEM
    // lanes) and columns kCols (w / 4) .. of the tile
    uint32_t it = 0, ci = 0, squares = 0;
    uint8_t* stage = smem + kOutOff + warp * kOutWarp;
    const int wr = warp & 3, wc = warp >> 2;
    // barrier of the epilogue warps; bounded like every wait, so that no warp is
    // left behind when another one has given up
    uint32_t phase = 0;
    auto together = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(esync);
      if (mbar_wait(esync, phase++ & 1, lim)) return true;
      report_error(err, YL_DEVERR_TIMEOUT);
      return false;
    };
    for (uint32_t k = 0;; ++k) {
      const int slot = k % kRing;
      if (!wait<PAIR>(&tfull[slot], (k / kRing) & 1, lim)) {
        report_error(err, YL_DEVERR_TIMEOUT);
        break;
      }
      const Ticket q = ring[slot];
      __syncwarp();
      if (lane == 0) arrive0(&tempty[slot]);
      if (q.mode == kNoTicket) break;
      const Item& im = t->it[q.item];
      const bool narrow = NARROW && (im.narrow >> q.mode & 1);
      const bool idle = narrow && wc != 0;  // 64 columns: the first four warps' alone
      if (u.muon && q.mode == UPDATE && q.step + 1 == steps.n) {
        // the parameter's rows towards L2 while the products run: a row of this
        // warp's columns per lane
        const long long r = (long long)(F::kSide * q.i + 2 * rank) * kBlk + wr * 32 + lane;
        const int c0 = narrow ? q.j * kBlk : F::kSide * q.j * kBlk + wc * kCols;
        const int c1 = min(c0 + kCols, im.cols);
        if (r < im.rows && !idle)
          for (int c = c0; c < c1; c += 32) prefetch_l2(im.dst + r * im.ldd + c);
      }
      float v[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) v[c] = 0.f;
      bool ok = true;
      // the accumulators of the ticket, as the MMA thread fills them
      for (int kb = 0; kb < q.nk; ++ci) {
        const bool fine = on_diagonal<PAIR, NARROW>(im, q, kb++);
        if (!fine && kb < q.nk && !on_diagonal<PAIR, NARROW>(im, q, kb)) ++kb;
        const int buf = ci % kAccs;
        if (!wait<PAIR>(&acc_full[buf], (ci / kAccs) & 1, lim)) {
          report_error(err, YL_DEVERR_TIMEOUT);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at =
            tmem + ((uint32_t)(wr * 32) << 16) + (uint32_t)(buf * F::kAccCols + wc * kCols);
        // 16 columns at a time (without PAIR those of hi hi, then those of the small
        // terms): the next read runs while this one is added
        constexpr int kReads = 128 / 16;
        const int small = narrow ? 64 : 128;
        auto col = [&](int p) { return PAIR ? p * 16 : (p >> 2) * small + (p & 3) * 16; };
        if (!idle) {
          uint32_t acc[2][16];
          tmem_ld_32x32b_x16(at, acc[0]);
#pragma unroll
          for (int p = 0; p < kReads; ++p) {
            tmem_ld_wait();
            if (p + 1 < kReads) tmem_ld_32x32b_x16(at + col(p + 1), acc[(p + 1) & 1]);
#pragma unroll
            for (int c = 0; c < 16; ++c)
              v[(PAIR ? p : p & 3) * 16 + c] += __uint_as_float(acc[p & 1][c]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive0(&acc_empty[buf]);
      }
      if (!ok) break;
      it += q.nk;
      if (q.mode == GRAM && im.ks > 1) {
        // leave this share's sum; the block that finishes a tile's last share adds
        // them all, in share order whoever that is
        // one block's part of a tile
        const size_t slice = (size_t)128 * (narrow ? 64 : F::kTile);
        const size_t slot0 = ((size_t)q.tile * F::kCtas + rank) * im.ks;
        float* part = im.partial + slot0 * slice + (size_t)(wc * kCols) * 128 + wr * 32 + lane;
        float* mine = part + (size_t)q.share * slice;
        if (!idle) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) __stcg(mine + c * 128, v[c]);
        }
        if (!together()) break;
        if (threadIdx.x == 0) {
          __threadfence();  // with the barrier: all of the block's stores
          const int seen = atomicAdd(
              t->ctrl + kCtrlSplit + im.split0 + q.tile * F::kCtas + (int)rank, 1);
          __threadfence();
          *last_share = seen == im.ks * (q.step + 1) - 1;
        }
        if (!together()) break;
        const bool mine_is_last = *last_share != 0;
        if (!mine_is_last) continue;  // thread 0 writes the flag again only behind a barrier
#pragma unroll
        for (int c = 0; c < kCols; ++c) v[c] = 0.f;
        for (int sh = 0; sh < (idle ? 0 : im.ks); ++sh) {
          const float* p = part + (size_t)sh * slice;
#pragma unroll
          for (int c = 0; c < kCols; ++c) v[c] += __ldcg(p + c * 128);
        }
      }
      const bool sq = q.mode != UPDATE, last = !sq && q.step + 1 == steps.n;
      const int rbt = sq ? im.mb : im.rb, cbt = sq ? im.mb : im.cb;
      // row block and row inside it
      const int rblk = F::kSide * q.i + 2 * rank + (wr >> 1), r64 = (wr & 1) * 32 + lane;
      const float c2 = q.c2;
      uint8_t* out = sq ? (q.mode == GRAM ? im.a : im.p) : im.x[(q.step & 1) ^ 1];
      const size_t plane = (size_t)rbt * cbt * kBlkBytes;
      const uint8_t* own = nullptr;  // this warp's 128 columns of the tile's own A
      if (q.mode == SQUARE) {
        const uint32_t e = it + (PAIR ? wc : 0);
        if (!mbar_wait(&full[e % kStages], (e / kStages) & 1, lim)) {
          report_error(err, YL_DEVERR_TIMEOUT);
          break;
        }
        own = smem + (e % kStages) * kStageBytes;
      }
#pragma unroll
      for (int slab = 0; slab < kCols / 64; ++slab) {
        const int cblk = narrow ? q.j : F::kSide * q.j + wc * (kCols / 64) + slab;
        if (idle || rblk >= rbt || cblk >= cbt) continue;  // uniform in the warp
        float* w = v + slab * 64;
#pragma unroll
        for (int c = 0; c < 64; ++c) w[c] *= c2;
        if (last) {
          // 32 rows x 32 columns through shared memory (columns rotated by the
          // row), then whole row pieces to the result
          float* st = reinterpret_cast<float*>(stage);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 32; ++c) st[lane * 32 + ((c + lane) & 31)] = w[half * 32 + c];
            __syncwarp();
            const long long r0 = (long long)rblk * kBlk + (wr & 1) * 32;
            const long long col = (long long)cblk * kBlk + half * 32 + lane;
            if (col < im.cols) {
              const int nr = (int)min(32LL, im.rows - r0);
              float* d = im.dst + r0 * im.ldd + col;
#pragma unroll 1
              for (int r1 = 0; r1 < nr; r1 += 16) {
                float pv[16];  // the parameter's rows are all on their way before the first is used
                if (u.muon) {
#pragma unroll
                  for (int r = 0; r < 16; ++r)
                    pv[r] = r1 + r < nr ? __ldcs(d + (r1 + r) * im.ldd) : 0.f;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  float x = st[(r1 + r) * 32 + ((lane + r1 + r) & 31)];
                  if (u.muon) x = pv[r] * (1.f - u.lr * u.decay) - u.lr * im.scale * x;
                  if (r1 + r < nr) __stcs(d + (r1 + r) * im.ldd, x);
                }
              }
            }
          }
          continue;
        }
        const size_t blk = ((size_t)rblk * cbt + cblk) * kBlkBytes;
        if (q.mode == SQUARE) {
          const float s1 = q.s1, s0 = steps.s0[q.step];
          const uint8_t* ah = own + (2 * (wr >> 1) + (PAIR ? slab : wc)) * kBlkBytes + r64 * 128;
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            const int at = (ch ^ (r64 & 7)) << 4;
            const uint4 h4 = *reinterpret_cast<const uint4*>(ah + at);
            const uint4 l4 = *reinterpret_cast<const uint4*>(ah + 2 * kOpBytes + at);
            const __half2* h = reinterpret_cast<const __half2*>(&h4);
            const __half2* l = reinterpret_cast<const __half2*>(&l4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 hf = __half22float2(h[j]), lf = __half22float2(l[j]);
              w[ch * 8 + 2 * j] += s1 * (hf.x + lf.x);
              w[ch * 8 + 2 * j + 1] += s1 * (hf.y + lf.y);
            }
          }
          if (rblk == cblk) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (r64 == c) w[c] += s0;
          }
        }
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {  // hi plane, then what is left of v as the lo plane
          if (lane == 0) bulk_wait_group_read<0>();  // the staging rows are free again
          __syncwarp();
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            __align__(16) __half2 h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float* x = w + ch * 8 + 2 * j;
              h[j] = __floats2half2_rn(x[0], x[1]);
              if (pl == 0) {
                const float2 f = __half22float2(h[j]);
                x[0] -= f.x;
                x[1] -= f.y;
              }
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((ch ^ (r64 & 7)) << 4)) =
                *reinterpret_cast<const uint4*>(h);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            bulk_store(out + blk + pl * plane + (wr & 1) * 4096, smem_u32(stage), 4096);
            bulk_commit_group();
          }
        }
      }
      if (last) continue;  // nothing waits for the results
      if (lane == 0) bulk_wait_group_all();
      // everything this block wrote of the tile is in memory before the count says so
      if (!together()) break;
      if (q.mode == SQUARE) {
        // freed once the tensor-core thread has passed them, long ago by now
        if (threadIdx.x < F::kCtas) {
          if (wait<PAIR>(&seen[squares & 1], (squares >> 1) & 1, lim))
            mbar_arrive(&empty[(it + threadIdx.x) % kStages]);
          else
            report_error(err, YL_DEVERR_TIMEOUT);
        }
        ++squares;
        it += F::kCtas;
      }
      if (threadIdx.x == 0) add_release(t->ctrl + kCtrlDone + 3 * q.item + q.mode, 1);
    }
    if (lane == 0) bulk_wait_group_all();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // neither block's barriers or operands are used any more
  if (warp == kEpiWarps + 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, kTmemCols);
    else tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------- short matrices
// Matrices with a shorter side of at most 128 stay on the chip: a cluster of
// blocks holds the pairs of X in shared memory, each block its share of the long
// side, from the first read of the input to the write of the result, and one
// launch does the norm, all steps and the update.  Per step each block multiplies
// its share of the Gram sum, the blocks exchange the sums by bulk copies between
// their shared memories (every block adds up a few rows in rank order and hands
// the finished rows to all), and each forms P for itself and updates its share.
constexpr int kChipBlocks = 6;                       // most 64 x 64 blocks of a block's share
constexpr int kChipShare = 16;                       // most blocks of a cluster
constexpr int kChipXPlane = kChipBlocks * kBlkBytes;
constexpr int kChipAOff = 2 * kChipXPlane;           // A, then P; before that the Gram sums
constexpr int kChipAPlane = 4 * kBlkBytes;
constexpr int kChipOutOff = kChipAOff + 2 * kChipAPlane;  // what the block sends
constexpr int kChipBarOff = kChipOutOff + 2 * kChipAPlane;
// barriers and norms, the factors of every step, alignment
constexpr int kChipFactors = 4;
constexpr int kChipSmem = kChipBarOff + 512 + kMaxSteps * kChipFactors * 4 + 1024;
static_assert(kChipSmem <= 227 * 1024, "a block's shared memory");
constexpr int kChipThreads = 256;

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// Sums the accumulators 0 .. n-1 of a warp's 32 rows x 64 columns.
__device__ __forceinline__ void sum_accumulators(uint32_t at, int n, float (&v)[64]) {
#pragma unroll
  for (int c = 0; c < 64; ++c) v[c] = 0.f;
#pragma unroll 1
  for (int a = 0; a < n; ++a) {
    uint32_t acc[2][16];
    tmem_ld_32x32b_x16(at + a * 128, acc[0]);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      tmem_ld_wait();
      if (p < 3) tmem_ld_32x32b_x16(at + a * 128 + (p + 1) * 16, acc[(p + 1) & 1]);
#pragma unroll
      for (int c = 0; c < 16; ++c) v[p * 16 + c] += __uint_as_float(acc[p & 1][c]);
    }
  }
}

// Eight values as a 16-byte chunk of either plane.
__device__ __forceinline__ void split8(const float* v, uint4* hi, uint4* lo) {
  __half2 h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    const float2 f = __half22float2(h[j]);
    l[j] = __floats2half2_rn(v[2 * j] - f.x, v[2 * j + 1] - f.y);
  }
  *hi = *reinterpret_cast<const uint4*>(h);
  *lo = *reinterpret_cast<const uint4*>(l);
}

__global__ void __launch_bounds__(kChipThreads, 1)
    ns_chip_kernel(const __grid_constant__ Table t, const __grid_constant__ Steps steps,
                   const __grid_constant__ Update u, float sx0, int share, int* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + kChipBarOff);
  uint64_t* sums_in = done + 1;   // other blocks' sums of this block's rows
  uint64_t* rows_in = done + 2;   // finished rows of A
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 3);
  double* norms = reinterpret_cast<double*>(smem + kChipBarOff + 64);  // [kChipShare]
  float* factors = reinterpret_cast<float*>(smem + kChipBarOff + 512);  // g2, s1, s2, u2 per step
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp & 3, wc = warp >> 2;
  const int rank = (int)cluster_rank();
  const Item& it = t.it[blockIdx.x / share];
  const bool tall = it.rows > it.cols;
  const int mb = it.mb, nb = max(it.rb, it.cb);
  const int w = (nb + share - 1) / share;  // blocks of a share
  const int first = rank * w, mw = max(0, min(w, nb - first));
  const long long lim = wait_limit(err);
  if (tid == 0) {
    mbar_init(done, 1);
    mbar_init(sums_in, 1);
    mbar_init(rows_in, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }

  // ---- the input: momentum step, norm, pairs.  A unit is 8 columns of a row;
  // a thread keeps all of its units in registers between the two.
  constexpr int kUnits = kChipBlocks * 64 * 8 / kChipThreads;
  float v[kUnits][8];
  const float clipf = u.muon ? clip_factor(u) : 1.f;
  // blocks of the share, in rows and in columns
  const int brows = tall ? mw : mb, bcols = tall ? mb : mw;
  const long long row0 = tall ? (long long)first * kBlk : 0;
  const long long col0 = tall ? 0 : (long long)first * kBlk;
  const int units = brows * kBlk * bcols * 8;
  double sq = 0.0;
#pragma unroll
  for (int e = 0; e < kUnits; ++e) {
    const int un = tid + e * kChipThreads;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[e][j] = 0.f;
    if (un >= units) continue;
    const int rr = un / (bcols * 8), cc = un - rr * bcols * 8;
    const long long r = row0 + rr, c = col0 + cc * 8;
    if (r >= it.rows || c >= it.cols) continue;
    const float* x = it.src + r * it.lds + c;
    const int n = (int)min(8LL, it.cols - c);
    float g[8], m[8];
    const bool vec = it.vec && n == 8;
    if (vec) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(x) + q);
        g[4 * q] = f.x, g[4 * q + 1] = f.y, g[4 * q + 2] = f.z, g[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = j < n ? __ldg(x + j) : 0.f;
    }
    if (!u.muon) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[e][j] = g[j];
      continue;
    }
    float* mo = it.mom + r * it.cols + c;
    if (vec) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 f = reinterpret_cast<const float4*>(mo)[q];
        m[4 * q] = f.x, m[4 * q + 1] = f.y, m[4 * q + 2] = f.z, m[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = j < n ? mo[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gv = clean(g[j], u, clipf);
      m[j] = u.mu * m[j] + gv;
      v[e][j] = j < n ? (u.nesterov ? gv + u.mu * m[j] : m[j]) : 0.f;
    }
    if (vec) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        reinterpret_cast<float4*>(mo)[q] =
            make_float4(m[4 * q], m[4 * q + 1], m[4 * q + 2], m[4 * q + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) mo[j] = m[j];
    }
  }
#pragma unroll
  for (int e = 0; e < kUnits; ++e)
#pragma unroll
    for (int j = 0; j < 8; ++j) sq += (double)v[e][j] * v[e][j];
  sq = block_sum256(sq);
  cluster_arrive();  // every block of the cluster runs: its shared memory can be written
  cluster_wait();
  if (tid < share) st_cluster_f64(map_to_rank(smem_u32(norms + rank), tid), sq);
  cluster_arrive();
  cluster_wait();
  double total = 0.0;
  for (int r = 0; r < share; ++r) total += norms[r];
  const int below = below_one(total, u.eps);
  double inv = inverse_norm(total, u.eps);
  if (below) inv = ldexp(inv, below);
  if (tid < steps.n) {
    const Lift lift(steps, below, tid);
    float* f = factors + kChipFactors * tid;
    f[0] = lift.gram(steps.g2[tid]);
    f[1] = lift.linear(steps.s1[tid]);
    f[2] = lift.square(steps.s2[tid]);
    f[3] = lift.update(steps, below, tid, steps.u2[tid]);
  }

  // Block (long, short) of the share: a wide X keeps its row blocks together (the
  // 128 rows of a K-major operand), a tall one its row blocks along the long side.
  // (Operands of 128 rows run into other blocks where there are fewer rows: what
  // comes of those stays in rows that nothing reads.)
  const int lmax = kChipBlocks / mb;
  auto xoff = [&](int lb, int sb) {
    return (uint32_t)((tall ? sb * lmax + lb : lb * mb + sb) * kBlkBytes);
  };
#pragma unroll
  for (int e = 0; e < kUnits; ++e) {
    const int un = tid + e * kChipThreads;
    if (un >= units) continue;
    const int rr = un / (bcols * 8), cc = un - rr * bcols * 8;
    const int rblk = rr >> 6, r = rr & 63, cblk = cc >> 3, ch = cc & 7;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)(v[e][j] * inv) * sx0;
    uint4 hi, lo;
    split8(x, &hi, &lo);
    uint8_t* at = smem + (tall ? xoff(rblk, cblk) : xoff(cblk, rblk)) + r * 128 + ((ch ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(at) = hi;
    *reinterpret_cast<uint4*>(at + kChipXPlane) = lo;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lanes = tmem + ((uint32_t)(wr * 32) << 16) + (uint32_t)(wc * 64);
  const uint32_t xs = smem_u32(smem), as = smem_u32(smem + kChipAOff);
  uint32_t waits = 0;

  // Products of `kks` 16-deep slices, `chain` to an accumulator; operand(kk) gives
  // the hi plane's two descriptors, the lo planes lie `lplane`, `rplane` bytes on.
  auto multiply = [&](int kks, int chain, uint32_t idesc, uint32_t lplane, uint32_t rplane,
                      auto descriptors) {
    fence_proxy_async_smem();  // shared memory written by this block's threads
    __syncthreads();
    if (tid == 0) {
      tc_fence_after();
      for (int k0 = 0, a = 0; k0 < kks; k0 += chain, ++a) {
        const int k1 = min(kks, k0 + chain);
#pragma unroll 1
        for (int part = 0; part < 3; ++part)  // lo hi, hi lo, hi hi
          for (int kk = k0; kk < k1; ++kk) {
            uint64_t ld, rd;
            descriptors(kk, &ld, &rd);
            ld += part == 0 ? lplane >> 4 : 0;
            rd += part == 1 ? rplane >> 4 : 0;
            umma_f16(tmem + a * 128, ld, rd, idesc, (part | (kk - k0)) != 0);
          }
      }
      umma_commit(done);
    }
    const uint32_t parity = waits++ & 1;
    if (!mbar_wait(done, parity, lim)) {
      // too slow for the caller's limit: say so, but let the products finish, since
      // they still read this block's shared memory
      report_error(err, YL_DEVERR_TIMEOUT);
      mbar_wait(done, parity);
    }
    tc_fence_after();
  };
  // accumulators are read again before the next multiply overwrites them
  auto drained = [&]() { tc_fence_before(); };

  // Waits for copies from other blocks; one that takes too long for the caller's
  // limit is reported and still waited for, since it writes to this block.
  auto arrived = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_wait_cluster(bar, parity, lim)) return;
    report_error(err, YL_DEVERR_TIMEOUT);
    mbar_wait_cluster(bar, parity);
  };
  const int rows = mb * kBlk / share;  // rows of A that a block adds up
  uint8_t* outbox = smem + kChipOutOff;
  for (int s = 0; s < steps.n; ++s) {
    const float* factor = factors + kChipFactors * s;
    // ---- this share of A = X X^T (X^T X)
    const int kks = 4 * mw, gchain = max(1, (kks + 3) / 4);
    if (kks > 0)
      multiply(kks, gchain, idesc_f16(128, mb * 64, tall, tall), kChipXPlane, kChipXPlane,
               [&](int kk, uint64_t* l, uint64_t* r) {
                 const uint32_t at = xs + xoff(kk >> 2, 0) + (kk & 3) * (tall ? 2048 : 32);
                 *l = *r = sw128_desc(at, tall ? lmax * kBlkBytes : 16, 1024);
               });
    float p[64];
    sum_accumulators(lanes, kks > 0 ? (kks + gchain - 1) / gchain : 0, p);
    drained();
    const int r64 = (wr & 1) * 32 + lane;  // this thread's row inside its block of A
    const bool in_a = wc < mb && (wr >> 1) < mb;
    uint8_t* a_row = smem + kChipAOff + (wc * 2 + (wr >> 1)) * kBlkBytes + r64 * 128;
    if (share == 1) {
      if (in_a) {
#pragma unroll
        for (int c = 0; c < 64; ++c) p[c] *= factor[0];
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint4 hi, lo;
          split8(p + ch * 8, &hi, &lo);
          uint8_t* at = a_row + ((ch ^ (r64 & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = hi;
          *reinterpret_cast<uint4*>(at + kChipAPlane) = lo;
        }
      }
    } else {
      // ---- sums to the blocks that add them up: rows of 64 mb floats, the block of
      // row r is r / rows; 16-byte pieces rotated by the row against bank conflicts
      const uint32_t pitch = mb * 256;
      if (s == 0) cluster_arrive();
      cluster_wait();  // no block needs its P any more, and all have what this one sent last
      if (in_a) {
        const int row = wr * 32 + lane;
        uint8_t* to = outbox + row * pitch + wc * 256;
#pragma unroll
        for (int q = 0; q < 16; ++q)
          *reinterpret_cast<float4*>(to + (((q + row) & 15) << 4)) =
              make_float4(p[4 * q], p[4 * q + 1], p[4 * q + 2], p[4 * q + 3]);
      }
      if (tid == 0) {
        mbar_arrive_expect_tx(sums_in, (uint32_t)(mb * kBlk) * pitch);
        mbar_arrive_expect_tx(rows_in, (uint32_t)(2 * mb * mb) * kBlkBytes);
      }
      fence_proxy_async_smem();
      __syncthreads();
      const uint32_t bytes = rows * pitch;  // to and from one block
      if (tid < share) {
        bulk_copy_cluster(map_to_rank(as + rank * bytes, tid),
                          smem_u32(outbox) + tid * bytes, bytes,
                          map_to_rank(smem_u32(sums_in), tid));
      }
      arrived(sums_in, s & 1);
      // ---- this block's rows, in rank order; a piece is 8 columns of a row
      uint4 hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = tid + i * kChipThreads, r = e / (8 * mb), c8 = e - r * 8 * mb;
        if (r >= rows) continue;
        const int row = rank * rows + r;
        const uint8_t* from = smem + kChipAOff + r * pitch + (c8 >> 3) * 256;
        const int q = 2 * (c8 & 7);
        float a[8] = {};
        for (int k = 0; k < share; ++k, from += bytes) {
          const float4 x = *reinterpret_cast<const float4*>(from + (((q + row) & 15) << 4));
          const float4 y = *reinterpret_cast<const float4*>(from + (((q + 1 + row) & 15) << 4));
          a[0] += x.x, a[1] += x.y, a[2] += x.z, a[3] += x.w;
          a[4] += y.x, a[5] += y.y, a[6] += y.z, a[7] += y.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] *= factor[0];
        split8(a, &hi[i], &lo[i]);
      }
      // ---- finished rows to every block: in both planes and each column block the
      // rows of a block lie together.  The outbox is free again once every block has
      // its sums, which the barrier says.
      fence_proxy_async_smem();
      cluster_arrive();
      cluster_wait();
      const uint32_t piece = rows * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = tid + i * kChipThreads, r = e / (8 * mb), c8 = e - r * 8 * mb;
        if (r >= rows) continue;
        uint8_t* to = outbox + (c8 >> 3) * piece + r * 128 +
                      (((c8 & 7) ^ ((rank * rows + r) & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = hi[i];
        *reinterpret_cast<uint4*>(to + mb * piece) = lo[i];
      }
      fence_proxy_async_smem();
      __syncthreads();
      const int row0a = rank * rows;
      for (int k = tid; k < share * 2 * mb; k += kChipThreads) {
        const int dst = k / (2 * mb), pl = (k / mb) & 1, cb = k % mb;
        const uint32_t at = as + pl * kChipAPlane + (cb * 2 + (row0a >> 6)) * kBlkBytes +
                            (row0a & 63) * 128;
        bulk_copy_cluster(map_to_rank(at, dst), smem_u32(outbox) + (pl * mb + cb) * piece, piece,
                          map_to_rank(smem_u32(rows_in), dst));
      }
      arrived(rows_in, s & 1);
    }
    // ---- P = s0 I + s1 A + s2 A A, over A
    multiply(4 * mb, mb, idesc_f16(128, mb * 64, 0, 0), kChipAPlane, kChipAPlane,
             [&](int kk, uint64_t* l, uint64_t* r) {
               *l = *r = sw128_desc(as + (kk >> 2) * 2 * kBlkBytes + (kk & 3) * 32, 16, 1024);
             });
    sum_accumulators(lanes, 4, p);
    drained();
    if (in_a) {
      const float s0 = steps.s0[s], s1 = factor[1], s2 = factor[2];
#pragma unroll
      for (int ch = 0; ch < 8; ++ch) {
        uint8_t* at = a_row + ((ch ^ (r64 & 7)) << 4);
        const uint4 h4 = *reinterpret_cast<const uint4*>(at);
        const uint4 l4 = *reinterpret_cast<const uint4*>(at + kChipAPlane);
        const __half2* h = reinterpret_cast<const __half2*>(&h4);
        const __half2* l = reinterpret_cast<const __half2*>(&l4);
        float o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 hf = __half22float2(h[j]), lf = __half22float2(l[j]);
          o[2 * j] = s2 * p[ch * 8 + 2 * j] + s1 * (hf.x + lf.x);
          o[2 * j + 1] = s2 * p[ch * 8 + 2 * j + 1] + s1 * (hf.y + lf.y);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (wc == (wr >> 1) && r64 == ch * 8 + j) o[j] += s0;
        uint4 a, b;
        split8(o, &a, &b);
        *reinterpret_cast<uint4*>(at) = a;
        *reinterpret_cast<uint4*>(at + kChipAPlane) = b;
      }
    }
    // ---- X' = P X (X P), two blocks of the long side at a time
    const bool last = s + 1 == steps.n;
    for (int hf = 0; 2 * hf < mw; ++hf) {
      const int hb = min(2, mw - 2 * hf);
      const uint32_t idesc =
          tall ? idesc_f16(128, mb * 64, 0, 0) : idesc_f16(128, hb * 64, 0, 1);
      multiply(4 * mb, mb, idesc, tall ? kChipXPlane : kChipAPlane, tall ? kChipAPlane : kChipXPlane,
               [&](int kk, uint64_t* l, uint64_t* r) {
                 const int sb = kk >> 2, q = kk & 3;
                 const uint64_t pd = sw128_desc(as + sb * 2 * kBlkBytes + q * 32, 16, 1024);
                 if (tall) {
                   *l = sw128_desc(xs + xoff(2 * hf, sb) + q * 32, 16, 1024);
                   *r = pd;
                 } else {
                   *l = pd;
                   *r = sw128_desc(xs + xoff(2 * hf, sb) + q * 2048, mb * kBlkBytes, 1024);
                 }
               });
      sum_accumulators(lanes, 4, p);
      drained();
      const int lrow = tall ? 2 * hf + (wr >> 1) : (wr >> 1);  // row and column block of the share
      const int lcol = tall ? wc : 2 * hf + wc;
      const bool inside = lrow < brows && lcol < bcols;
      const float c2 = factor[3];
      if (inside) {
#pragma unroll
        for (int c = 0; c < 64; ++c) p[c] *= c2;
      }
      if (!last) {
        if (inside) {
          uint8_t* blk = smem + (tall ? xoff(lrow, lcol) : xoff(lcol, lrow)) + r64 * 128;
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            uint4 a, b;
            split8(p + ch * 8, &a, &b);
            uint8_t* at = blk + ((ch ^ (r64 & 7)) << 4);
            *reinterpret_cast<uint4*>(at) = a;
            *reinterpret_cast<uint4*>(at + kChipXPlane) = b;
          }
        }
        continue;
      }
      // the result, 32 rows x 32 columns at a time through this half's own blocks
      if (inside) {
        float* st = reinterpret_cast<float*>(
            smem + (tall ? xoff(2 * hf, wc) + wr * 4096 : xoff(2 * hf + wc, 0) + wr * 4096));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 32; ++c) st[lane * 32 + ((c + lane) & 31)] = p[half * 32 + c];
          __syncwarp();
          const long long r0 = row0 + lrow * kBlk + (wr & 1) * 32;
          const long long col = col0 + lcol * kBlk + half * 32 + lane;
          if (col < it.cols) {
            const int nr = (int)max(0LL, min(32LL, it.rows - r0));
            float* d = it.dst + r0 * it.ldd + col;
#pragma unroll 1
            for (int r1 = 0; r1 < nr; r1 += 16) {
              float pv[16];
              if (u.muon) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                  pv[r] = r1 + r < nr ? __ldcs(d + (r1 + r) * it.ldd) : 0.f;
              }
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                float x = st[(r1 + r) * 32 + ((lane + r1 + r) & 31)];
                if (u.muon) x = pv[r] * (1.f - u.lr * u.decay) - u.lr * it.scale * x;
                if (r1 + r < nr) __stcs(d + (r1 + r) * it.ldd, x);
              }
            }
          }
        }
      }
    }
    __syncthreads();
    // this block's P may be overwritten; waited for in the next step
    if (share > 1) cluster_arrive();
  }
  if (share > 1) cluster_wait();  // no block leaves while another may still write to it
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------- host side
long long update_tiles(const Item& it, int side_rows, int side_cols) {
  const long long rb = (it.rows + kBlk - 1) / kBlk, cb = (it.cols + kBlk - 1) / kBlk;
  return (rb + side_rows - 1) / side_rows * ((cb + side_cols - 1) / side_cols);
}
// Tiles on and below the diagonal of A and P.
long long lower_tiles(const Item& it, int side, bool narrow) {
  const long long mb = (std::min(it.rows, it.cols) + kBlk - 1) / kBlk, mt = (mb + side - 1) / side;
  return narrow ? mt * (mt + 1) - (mb & 1) : mt * (mt + 1) / 2;
}

// 64-deep k-blocks of a tile's sum in SQUARE and UPDATE.
int k_blocks(const Item& it) { return (std::min(it.rows, it.cols) + kBlk - 1) / kBlk; }
// Thousands of cycles for a k-block.
double block_time(bool narrow) { return narrow ? 0.8 : 1.1; }
// Shares of GRAM's long side, at most `most`: the number with the shortest way
// through a tile.  The sums' way through memory takes 5k cycles, and 1.2k more for
// each share that the last block reads.
int shares(const Item& it, bool narrow, int most, double* time) {
  const int nk = (std::max(it.rows, it.cols) + kBlk - 1) / kBlk;
  int best = 1;
  double before = HUGE_VAL;
  *time = block_time(narrow) * nk;
  for (int ks = 2; ks <= std::min(most, nk); ++ks) {
    const double cost = block_time(narrow) * nk / ks + 5 + 1.2 * ks;
    if (cost > before) break;  // it only grows from here
    if (cost < *time) *time = cost, best = ks;
    before = cost;
  }
  return best;
}
// Thousands of cycles for a tile of a phase (about 9 beside its products), and the
// tiles' number.
double tile_time(const Item& it, int mode, bool narrow, long long* tiles) {
  if (mode == UPDATE) *tiles = update_tiles(it, 2, narrow ? 1 : 2);
  else *tiles = lower_tiles(it, 2, narrow);
  double products = block_time(narrow) * k_blocks(it);
  if (mode == GRAM) *tiles *= shares(it, narrow, kMaxShares, &products);
  return 9 + products;
}

// Tiles of 64 columns for a phase's longest products, as far as the longest one
// gets shorter and the SMs still hold them all (512 x 512 166 -> 146 us, 1024 x 1024
// 238 -> 219 us; with those of GRAM and SQUARE alone 512 x 4608 221 -> 203 us).  Not
// where the phases of many matrices overlap and leave no SM idle: the U-Net's table
// took 460 us so, 451 without.
void choose_narrow(Table* t, int num_sms) {
  for (int k = 0; k < t->count; ++k) t->it[k].narrow = 0;
  if (t->pair || t->chip) return;
  for (int mode = 2; mode >= 0; --mode) {
    int order[kMaxItems];
    double time[kMaxItems][2], total[kMaxItems][2], all = 0;
    for (int k = 0; k < t->count; ++k) {
      order[k] = k;
      for (int narrow = 0; narrow < 2; ++narrow) {
        long long tiles;
        time[k][narrow] = tile_time(t->it[k], mode, narrow, &tiles);
        total[k][narrow] = time[k][narrow] * tiles;
      }
      all += total[k][0];
    }
    std::sort(order, order + t->count, [&](int x, int y) {
      return time[x][0] != time[y][0] ? time[x][0] > time[y][0] : x < y;
    });
    if (mode == UPDATE && t->count > 1 && all > time[order[0]][0] * num_sms) return;
    double best = std::max(time[order[0]][0], all / num_sms), longest = 0;
    int chosen = 0;
    for (int n = 1; n <= t->count; ++n) {
      const int k = order[n - 1];
      all += total[k][1] - total[k][0];
      longest = std::max(longest, time[k][1]);
      const double rest = n < t->count ? time[order[n]][0] : 0.0;
      const double now = std::max({longest, rest, all / num_sms});
      if (now < best) best = now, chosen = n;
    }
    for (int n = 0; n < chosen; ++n) t->it[order[n]].narrow |= 1 << mode;
  }
}

// Sizes the table's workspace, or (with a base address) places it; returns the
// bytes it takes.
size_t place(Table* t, int num_sms, char* ws) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = ws + off;
    off += (bytes + 1023) & ~(size_t)1023;
    return (uint8_t*)p;
  };
  take(sizeof(Table));
  for (int k = 0; k < t->count; ++k) {
    Item& it = t->it[k];
    auto blocks = [](int v) { return (v + kBlk - 1) / kBlk; };
    it.rb = blocks(it.rows);
    it.cb = blocks(it.cols);
    it.mb = std::min(it.rb, it.cb);
    const long long n = (long long)it.rows * it.cols;
    it.chunk = (int)((n / kNormParts + kNormChunk) / kNormChunk * kNormChunk);
    it.chunks = (int)((n + it.chunk - 1) / it.chunk);
    it.vec = !(((uintptr_t)it.src | (uintptr_t)it.mom | (uintptr_t)(it.lds * 4)) & 15);
    const size_t xb = (size_t)2 * it.rb * it.cb * kBlkBytes;
    const size_t mb = (size_t)2 * it.mb * it.mb * kBlkBytes;
    it.x[0] = take(xb);
    it.x[1] = take(xb);
    it.a = take(mb);
    it.p = take(mb);
    it.part = (double*)take(it.chunks * sizeof(double));
  }
  // Shares of GRAM's long side: at most as many as bring its tickets down to the
  // average per SM.
  auto nk = [](const Item& it) { return std::max(it.rb, it.cb); };
  const int ctas = t->pair ? 2 : 1, workers = num_sms / ctas;
  auto gram_tiles = [&](const Item& it) {
    return (int)lower_tiles(it, 2 * ctas, it.narrow >> GRAM & 1);
  };
  double kb = 0;
  for (int k = 0; k < t->count; ++k) kb += (double)gram_tiles(t->it[k]) * nk(t->it[k]);
  const double fair = kb / workers;
  int splits = 0;
  for (int k = 0; k < t->count; ++k) {
    Item& it = t->it[k];
    double time;
    it.ks = shares(it, it.narrow >> GRAM & 1,
                   (int)std::min(std::round(nk(it) / std::max(fair, 1.0)), (double)kMaxShares), &time);
    it.split0 = splits;
    it.partial = nullptr;
    if (it.ks > 1) {
      splits += gram_tiles(it) * ctas;
      const size_t tile = (size_t)128 * ctas * 128 * ctas * sizeof(float);
      it.partial = (float*)take(gram_tiles(it) * it.ks * tile);
    }
  }
  t->ctrl_ints = kCtrlSplit + splits;
  t->ctrl = (int*)take(t->ctrl_ints * sizeof(int));
  return off;
}

struct Schedule {
  int steps;
  float q[3 * kMaxSteps];    // coefficients
  double sx[kMaxSteps + 1];  // scales of X before each step and at the end, powers of two
  double sa[kMaxSteps], sp[kMaxSteps];
  int rise[kMaxSteps + 1];   // see Steps
};

// Coefficients with the scales of the pairs folded in, and half of what the tensor
// core's truncation takes off the products of dense matrices.
Steps scaled_steps(const Schedule& s) {
  Steps st;
  st.n = s.steps;
  std::copy(s.rise, s.rise + s.steps + 1, st.rise);
  for (int k = 0; k < s.steps; ++k) {
    const double sx = s.sx[k], sa = s.sa[k], sp = s.sp[k], back = 1.0 + 0x1p-23;
    st.g2[k] = (float)(sa / (sx * sx) * back);
    st.s0[k] = (float)(s.q[3 * k] * sp);
    st.s1[k] = (float)(s.q[3 * k + 1] * sp / sa);
    st.s2[k] = (float)(s.q[3 * k + 2] * sp / (sa * sa) * back);
    st.u2[k] = (float)((k + 1 == s.steps ? 1.0 : s.sx[k + 1]) / (sp * sx));
  }
  return st;
}

// Whether a matrix can stay on the chip, in a cluster of at most `largest` blocks.
bool on_chip(const Item& it, int largest) {
  const int m = std::min(it.rows, it.cols), n = std::max(it.rows, it.cols);
  const int mb = (m + kBlk - 1) / kBlk, nb = (n + kBlk - 1) / kBlk;
  return mb <= 2 && nb <= largest * (kChipBlocks / mb);
}

cudaLaunchConfig_t chip_config(int matrices, int share, cudaLaunchAttribute* cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(matrices * share);
  cfg.blockDim = dim3(kChipThreads);
  cfg.dynamicSmemBytes = kChipSmem;
  cluster->id = cudaLaunchAttributeClusterDimension;
  cluster->val.clusterDim.x = share;
  cluster->val.clusterDim.y = cluster->val.clusterDim.z = 1;
  cfg.attrs = cluster;
  cfg.numAttrs = 1;
  return cfg;
}

// The largest cluster of the on-chip kernel that this device, or the part of it that
// the process has, finds room for (0: none); asked once per context.
int largest_cluster(yl_ctx* ctx) {
  if (ctx->chip_cluster >= 0) return ctx->chip_cluster;
  int largest = 0;
  if (cudaFuncSetAttribute(ns_chip_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kChipSmem) ==
          cudaSuccess &&
      cudaFuncSetAttribute(ns_chip_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) ==
          cudaSuccess) {
    for (int share = kChipShare; share > 0 && largest == 0; share /= 2) {
      cudaLaunchAttribute cluster;
      const cudaLaunchConfig_t cfg = chip_config(1, share, &cluster);
      int room = 0;
      if (cudaOccupancyMaxActiveClusters(&room, ns_chip_kernel, &cfg) == cudaSuccess && room > 0)
        largest = share;
    }
  }
  cudaGetLastError();  // sizes that do not fit are no error of this call
  return ctx->chip_cluster = largest;
}

// Blocks that the longest of these matrices needs for its share to fit.
int least_share(const Item* items, int count) {
  int share = 1;
  for (int k = 0; k < count; ++k) {
    const int rb = (items[k].rows + kBlk - 1) / kBlk, cb = (items[k].cols + kBlk - 1) / kBlk;
    while (share * (kChipBlocks / std::min(rb, cb)) < std::max(rb, cb)) share *= 2;
  }
  return share;
}

yl_status run_chip(yl_ctx* ctx, Table& t, const Update& u, const Schedule& s) {
  place(&t, ctx->num_sms, nullptr);  // sizes only: nothing of these is in the workspace
  // as many blocks to a matrix as its long side needs, and more while SMs are idle
  int longest = 0, share = least_share(t.it, t.count);
  for (int k = 0; k < t.count; ++k) longest = std::max({longest, t.it[k].rb, t.it[k].cb});
  // (clusters of 16 find room for only a few of themselves)
  while (share < longest && 2 * share * t.count <= (share < 8 ? 1.0 : 0.5) * ctx->num_sms &&
         2 * share <= largest_cluster(ctx))
    share *= 2;
  YL_CUDA(cudaFuncSetAttribute(ns_chip_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kChipSmem));
  if (share > 8)
    YL_CUDA(cudaFuncSetAttribute(ns_chip_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute cluster;
  cudaLaunchConfig_t cfg = chip_config(t.count, share, &cluster);
  cfg.stream = ctx->stream;
  YL_CUDA(cudaLaunchKernelEx(&cfg, ns_chip_kernel, t, scaled_steps(s), u, (float)s.sx[0], share,
                             ctx->dev_err));
  return check_launch("ns_chip_kernel");
}

yl_status run_table(yl_ctx* ctx, Table& t, const Update& u, const Schedule& s, char* ws) {
  if (t.chip) return run_chip(ctx, t, u, s);
  place(&t, ctx->num_sms, ws);
  const int ctas = t.pair ? 2 : 1, side = 2 * ctas;
  for (int m = 0; m < 3; ++m) t.tiles[m][0] = 0;
  t.blocks[0] = t.chunks[0] = 0;
  for (int k = 0; k < t.count; ++k) {
    const Item& it = t.it[k];
    auto narrow = [&](int mode) { return (it.narrow >> mode & 1) != 0; };
    t.tiles[GRAM][k + 1] = t.tiles[GRAM][k] + (int)lower_tiles(it, side, narrow(GRAM)) * it.ks;
    t.tiles[SQUARE][k + 1] = t.tiles[SQUARE][k] + (int)lower_tiles(it, side, narrow(SQUARE));
    t.tiles[UPDATE][k + 1] =
        t.tiles[UPDATE][k] + (int)update_tiles(it, side, narrow(UPDATE) ? 1 : side);
    t.blocks[k + 1] = t.blocks[k] + it.rb * it.cb;
    t.chunks[k + 1] = t.chunks[k] + it.chunks;
  }
  Table* dt = (Table*)ws;
  ns_norm_kernel<<<t.chunks[t.count], 256, 0, ctx->stream>>>(t, u, dt);
  YL_TRY(check_launch("ns_norm_kernel"));
  if (s.steps == 0) {
    ns_direct_kernel<<<t.chunks[t.count], 256, 0, ctx->stream>>>(dt, u);
    return check_launch("ns_direct_kernel");
  }
  ns_split_kernel<<<t.blocks[t.count], 256, 0, ctx->stream>>>(dt, u, (float)s.sx[0], dt->below);
  YL_TRY(check_launch("ns_split_kernel"));
  const Steps st = scaled_steps(s);
  // More blocks than a phase has tickets: they hold tickets of the phases to come,
  // so that no block is handed two of one phase (512 x 128 and 512 x 512 in 22
  // blocks, the most tickets of a phase: 291 us).
  long long tickets = 0;
  for (int m = 0; m < 3; ++m) tickets += (long long)s.steps * t.tiles[m][t.count];
  const int workers = (int)std::min<long long>(tickets, ctx->num_sms / ctas);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(workers * ctas);
  cfg.blockDim = dim3(kProductThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = 2;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = t.pair ? 1 : 0;
  bool narrow = false;
  for (int k = 0; k < t.count; ++k) narrow |= t.it[k].narrow != 0;
  auto kernel = t.pair   ? ns_steps_kernel<true, false>
                : narrow ? ns_steps_kernel<false, true>
                         : ns_steps_kernel<false, false>;
  YL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  YL_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const Table*)dt, st, u, ctx->dev_err));
  return check_launch("ns_steps_kernel");
}

// About how long a step of these matrices takes (us), by single blocks or by pairs
// of them on SMs that are all busy: 0.72 us a k-block of a 128 x 128 tile, 1.1 us of
// a 256 x 256 tile, and 2 and 6 us beside them.  The tiles of a single matrix go in
// whole waves; those of several fill one another's, and take at least one tile of
// each phase.
double step_time(const std::vector<const Item*>& items, int num_sms, bool pair) {
  const int side = pair ? 4 : 2, workers = pair ? num_sms / 2 : num_sms;
  const double block = pair ? 1.1 : 0.72, rest = pair ? 6 : 2;
  double sum = 0, chain = 0;
  for (const Item* it : items) {
    const double lower = (double)lower_tiles(*it, side, false);
    const double update = (double)update_tiles(*it, side, side);
    const double one = block * k_blocks(*it) + rest;
    const double nk = (std::max(it->rows, it->cols) + kBlk - 1) / kBlk;
    const double gram = block * nk + rest;
    if (items.size() > 1) {
      sum += (lower * gram + lower * one + update * one) / workers;
      chain = std::max(chain, 3 * one);
      continue;
    }
    // a Gram product that leaves SMs idle is shared out among them
    sum += lower < workers ? std::min(gram, lower * block * nk / workers + rest + 5)
                           : std::ceil(lower / workers) * gram;
    // half as wide tiles, each sooner done, while they fit
    const bool narrow = !pair && 2 * lower <= workers;
    sum += std::ceil(lower / workers) * (narrow ? 0.7 * one : one);
    sum += std::ceil(update / workers) * one;
  }
  return std::max(sum, chain);
}

// The tables of a call: matrices for pairs of blocks first, then the others.
// A pair does twice the products per shared-memory read, but has half as many and
// larger tiles to share among the SMs, so it pays where those stay full: 4096 x 4096
// 3.76 ms in pairs and 4.30 alone, 2560 x 2560 1.07 and 1.17, 8 of 1024 x 1024 0.59
// and 0.63, but 4 of them 0.41 and 0.34, 2048 x 2048 0.63 and 0.60, 1024 x 8192
// 0.61 and 0.57, 16 of 600 x 2400, which 256 x 256 tiles pad, 1.22 and 1.05.  (The estimates are within some
// 6% of that: pairs have to promise as much.)  Sides under kPairSide are mostly
// padding.  Where other matrices remain, they take a launch of their own.
template <class Fn>
yl_status for_tables(yl_ctx* ctx, const std::vector<Item>& items, int steps, Fn fn) {
  auto wide = [](const Item& it) { return std::min(it.rows, it.cols) >= kPairSide; };
  std::vector<const Item*> large;
  double others = 0;
  for (const Item& it : items) {
    if (wide(it)) large.push_back(&it);
    else others = std::max(others, 3 * (4.5 + 0.43 * k_blocks(it)));
  }
  const bool pairs = !large.empty() && step_time(large, ctx->num_sms, true) + others <
                                           0.94 * step_time(large, ctx->num_sms, false);
  // With longer matrices beside them the short ones cost the steps kernel less
  // than a launch of their own, and so do more clusters than the SMs hold at once
  // (24 of 128 x 1152: 267 us in clusters of 8, 168 us in the steps kernel; 14 of
  // them 138 and 158 us).
  const int largest = largest_cluster(ctx);
  const bool chip = steps > 0 &&
                    std::all_of(items.begin(), items.end(),
                                [&](const Item& it) { return on_chip(it, largest); }) &&
                    (long long)items.size() * least_share(items.data(), (int)items.size()) <=
                        ctx->num_sms;
  // Where the tiles of a phase nearly all find an SM at once, the longest chains of
  // products come first: what has to wait is then short (five odd shapes 245 -> 233
  // us).  Longer tables keep the caller's order (39 of the U-Net's 436 us,
  // sorted 446).
  std::vector<const Item*> order;
  double all = 0, longest = 0;
  for (const Item& it : items) {
    order.push_back(&it);
    long long tiles;
    const double time = tile_time(it, UPDATE, false, &tiles);
    all += time * tiles;
    longest = std::max(longest, time);
  }
  if (all <= longest * ctx->num_sms)
    std::sort(order.begin(), order.end(), [](const Item* x, const Item* y) {
      const int sx = k_blocks(*x), sy = k_blocks(*y);
      return sx != sy ? sx > sy : x < y;
    });
  auto t = std::make_unique<Table>();
  t->chip = chip;
  for (int pair = 1; pair >= 0; --pair) {
    t->count = 0;
    t->pair = pair;
    for (size_t k = 0; k <= items.size(); ++k) {
      if (t->count == kMaxItems || (k == items.size() && t->count > 0)) {
        choose_narrow(t.get(), ctx->num_sms);
        YL_TRY(fn(*t));
        t->count = 0;
      }
      if (k < items.size() && (pairs && wide(*order[k])) == (pair != 0))
        t->it[t->count++] = *order[k];
    }
  }
  return YL_OK;
}
// One table after the other, in the same workspace.
yl_status run_items(yl_ctx* ctx, const std::vector<Item>& items, const Update& u,
                    const Schedule& s, char* ws) {
  return for_tables(ctx, items, s.steps,
                    [&](Table& t) { return run_table(ctx, t, u, s, ws); });
}
size_t items_bytes(yl_ctx* ctx, const std::vector<Item>& items, int steps) {
  size_t most = 0;
  for_tables(ctx, items, steps, [&](Table& t) {
    if (!t.chip) most = std::max(most, place(&t, ctx->num_sms, nullptr));
    return YL_OK;
  });
  return most;
}

size_t norm_parts(long long n) { return (size_t)((n + kNormChunk - 1) / kNormChunk); }

constexpr float kQuintic[3] = {3.4445f, -4.7750f, 2.0315f};

// Largest power of two that keeps values up to `top` under fp16's 65504 with
// room for rounding.  (What steps have shrunk below kMinTop is at the end of fp32's
// range.)
constexpr double kMinTop = 0x1p-100;
double scale_for(double top) {
  int e;
  std::frexp(32768.0 / std::max(top, kMinTop), &e);
  return std::ldexp(1.0, e - 1);
}

// How far the steps may let a small singular value grow against the largest one.
// What lies under the pairs' floor is lost at the start of a step and grows from
// there on; where the small values are those of small rows, fp32 products would have
// kept it.  By a CPU model of the formats, rows of 1 and 1e-6 to 1e-10 by turns, 512 x
// 1024: 9 quintic steps (2^16.1) end 1.5e-6 off where fp32 products end 3.0e-6 off, 10
// (2^17.8) 4.7e-6 [3.5e-6], 12 (2^21.4) 5.4e-5, 20 (2^35.7) 2.8e-2.
constexpr double kMaxGrowth = 131072.0;

// The coefficients and scales of every step, if the coefficients keep the
// singular values (at most 1 at the start) below kMaxSigma and the growth of small
// ones below kMaxGrowth.
yl_status plan_steps(const char* who, int steps, const float* given, Schedule* s_out) {
  float* out = s_out->q;
  s_out->steps = steps;
  YL_CHECK(steps >= 0 && steps <= kMaxSteps, YL_ERR_INVALID, "%s: %d steps (0 to %d)", who, steps,
           kMaxSteps);
  double top = 1.0, growth = 1.0;
  s_out->rise[0] = 0;
  for (int s = 0; s < steps; ++s) {
    const float* q = given ? given + 3 * s : kQuintic;
    for (int i = 0; i < 3; ++i) {
      YL_CHECK(std::isfinite(q[i]), YL_ERR_INVALID, "%s: coefficient %d of step %d is not finite",
               who, i, s);
      out[3 * s + i] = q[i];
    }
    // |p| on [0, top] is largest at its end or where p' = 5 c t^2 + 3 b t + a = 0 with
    // t = s^2; the roots without a difference of nearly equal numbers
    const double a = q[0], b = q[1], c = q[2];
    auto p = [&](double v) { return std::fabs(v * (a + v * v * (b + v * v * c))); };
    double next = p(top);
    auto at = [&](double sq) {
      if (sq > 0 && sq < top * top) next = std::max(next, p(std::sqrt(sq)));
    };
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      const double r = -0.5 * (3 * b + std::copysign(std::sqrt(d), b));
      if (c != 0.0) at(r / (5 * c));
      if (r != 0.0) at(a / r);
    }
    const double inner = std::fabs(a) + std::fabs(b) * top * top + std::fabs(c) * top * top * top * top;
    YL_CHECK(next <= kMaxSigma && inner <= 1024.0, YL_ERR_UNSUPPORTED,
             "%s: the coefficients of step %d let singular values grow to %.3g (at most %.3g)", who,
             s, next, kMaxSigma);
    // entries of X are bounded by its largest singular value, those of A by its
    // square, those of P by inner
    s_out->sx[s] = scale_for(top);
    s_out->sa[s] = scale_for(top * top);
    s_out->sp[s] = scale_for(inner);
    // |p(s)| / s is largest at an end of [0, top] or where its derivative is 0
    auto gain = [&](double sq) { return std::fabs(a + sq * (b + sq * c)); };
    double most = std::max(gain(0.0), gain(top * top));
    if (c != 0.0) most = std::max(most, gain(std::min(top * top, std::max(0.0, -b / (2 * c)))));
    const double bound = std::max(next, kMinTop);  // what the next scale allows for
    const double up = most * top / bound;
    s_out->rise[s + 1] = s_out->rise[s] + (up > 1.0 ? (int)std::ceil(std::log2(up)) : 0);
    growth = std::max(growth, 1.0) * up;
    YL_CHECK(growth <= kMaxGrowth, YL_ERR_UNSUPPORTED,
             "%s: by step %d the coefficients let small singular values grow by %.3g against the "
             "largest (at most %.3g)",
             who, s, growth, kMaxGrowth);
    top = next;
  }
  s_out->sx[std::max(steps, 0)] = scale_for(top);
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
  if (rows_a == 1) lda = ldb;  // (a single row has no stride)
  if (rows_b == 1) ldb = lda;
  if (lda != ldb) return true;
  // columns of one buffer side by side?  (b - a) modulo the row stride
  long long d = ((long long)(b0 - a0) / 4) % lda;
  if (d < 0) d += lda;
  return !(d >= cols_a && d + cols_b <= lda);
}

yl_status check_steps(const char* who, int steps, const float* coeffs) {
  Schedule q;
  return plan_steps(who, steps, coeffs, &q);
}

yl_status newton_schulz(yl_ctx* ctx, const yl_ns_matrix* table, int count, int steps,
                        const float* coeffs, float eps) {
  const char* who = "yl_newton_schulz";
  Schedule q;
  YL_TRY(plan_steps(who, steps, coeffs, &q));
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
  // every result against every matrix whose extent meets its own
  struct Extent { const float *p, *end; long long ld; const Item* it; bool out; };
  std::vector<Extent> ext;
  for (const Item& it : items)
    for (int out = 0; out < 2; ++out) {
      const float* p = out ? it.dst : it.src;
      const long long ld = out ? it.ldd : it.lds;
      ext.push_back({p, p + (it.rows - 1) * ld + it.cols, ld, &it, out != 0});
    }
  std::sort(ext.begin(), ext.end(), [](const Extent& x, const Extent& y) { return x.p < y.p; });
  for (size_t i = 0; i < ext.size(); ++i)
    for (size_t j = i + 1; j < ext.size() && ext[j].p < ext[i].end; ++j) {
      const Extent &x = ext[i], &y = ext[j];
      if (!x.out && !y.out) continue;
      if (x.it == y.it && x.p == y.p && x.ld == y.ld) continue;  // in place
      YL_CHECK(!rows_overlap(x.p, x.ld, x.it->rows, x.it->cols, y.p, y.ld, y.it->rows, y.it->cols),
               YL_ERR_INVALID, "%s: a result overlaps another matrix of the table", who);
    }
  if (items.empty()) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  Update u{};
  u.eps = eps;
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, items_bytes(ctx, items, q.steps), &ws));
  YL_TRY(run_items(ctx, items, u, q, ws));
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
  Schedule q;
  YL_TRY(plan_steps(who, st.steps, coeffs, &q));
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
  YL_CHECK(!((uintptr_t)norm_out & 3), YL_ERR_INVALID,
           "%s: norm_out_dev is not a multiple of 4 bytes", who);
  if (norm_out) r.push_back({(uintptr_t)norm_out, (uintptr_t)(norm_out + 1), true});
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
  uintptr_t end = 0, wend = 0;  // behind every range so far, and every written one
  for (const Range& x : r) {
    YL_CHECK(!(x.lo < wend || (x.write && x.lo < end)), YL_ERR_INVALID,
             "%s: a parameter, a momentum or the norm overlaps another tensor", who);
    end = std::max(end, x.hi);
    if (x.write) wend = std::max(wend, x.hi);
  }
  const bool measure = norm_out || (st.clip_max_norm > 0.f && !norm);
  if (items.empty() && !measure) return YL_OK;
  DeviceGuard dev(ctx->device);
  YL_CUDA(dev.status());
  size_t parts = 0;
  if (measure) {
    for_tables(ctx, items, st.steps, [&](Table& t) {
      place(&t, ctx->num_sms, nullptr);
      for (int k = 0; k < t.count; ++k) parts += t.it[k].chunks;
      return YL_OK;
    });
  }
  ScratchCarver carve;
  const size_t o_norm = carve.take(sizeof(float)), o_parts = carve.take(parts * sizeof(double));
  carve.offset = (carve.offset + 1023) & ~(size_t)1023;
  const size_t o_items = carve.take(items_bytes(ctx, items, q.steps));
  Workspace work;
  char* ws = nullptr;
  YL_TRY(work.get(ctx, carve.offset, &ws));
  if (measure) {
    double* part = (double*)(ws + o_parts);
    float* out = norm_out ? norm_out : (float*)(ws + o_norm);
    YL_TRY(for_tables(ctx, items, st.steps, [&](Table& t) -> yl_status {
      place(&t, ctx->num_sms, nullptr);
      t.chunks[0] = 0;
      for (int k = 0; k < t.count; ++k) t.chunks[k + 1] = t.chunks[k] + t.it[k].chunks;
      table_square_kernel<<<t.chunks[t.count], 256, 0, ctx->stream>>>(t, st.grad_scale, st.sanitize,
                                                                     part);
      part += t.chunks[t.count];
      return check_launch("table_square_kernel");
    }));
    grad_norm_final_kernel<<<1, 256, 0, ctx->stream>>>((const double*)(ws + o_parts),
                                                       (long long)parts, out);
    YL_TRY(check_launch("grad_norm_final_kernel"));
    if (!norm) norm = out;
  }
  Update u{};
  u.muon = 1, u.nesterov = st.nesterov, u.sanitize = st.sanitize;
  u.mu = st.momentum, u.lr = st.lr, u.decay = st.weight_decay, u.grad_scale = st.grad_scale;
  u.clip = st.clip_max_norm, u.eps = st.eps, u.norm = norm;
  YL_TRY(run_items(ctx, items, u, q, ws + o_items));
  return work.done();
}

}  // namespace yl

using namespace yl;

extern "C" {

yl_status yl_debug_cluster_limit(yl_ctx* ctx, int blocks) {
  YL_CHECK(ctx, YL_ERR_INVALID, "yl_debug_cluster_limit: ctx is NULL");
  YL_CHECK(blocks >= -1 && blocks <= kChipShare && (blocks < 1 || (blocks & (blocks - 1)) == 0),
           YL_ERR_INVALID, "yl_debug_cluster_limit: %d blocks (-1, 0 or a power of two up to %d)",
           blocks, kChipShare);
  ctx->chip_cluster = blocks;
  return YL_OK;
}

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
