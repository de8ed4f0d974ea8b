// yl_internal.h -- shared host-side plumbing of the backend: status/error
// reporting, the context object, stream-ordered scratch memory.
#pragma once
#include <cuda_runtime.h>

#include <chrono>
#include <cstdarg>
#include <cstddef>
#include <cstdint>

#include "yume_c.h"

namespace yl {

// Records `msg` as this thread's last error and returns `st`.
yl_status set_error(yl_status st, const char* fmt, ...);

#define YL_CUDA(expr)                                                                      \
  do {                                                                                     \
    cudaError_t e_ = (expr);                                                               \
    if (e_ != cudaSuccess)                                                                 \
      return ::yl::set_error(YL_ERR_CUDA, "%s failed: %s (%s:%d)", #expr,                  \
                             cudaGetErrorString(e_), __FILE__, __LINE__);                  \
  } while (0)

#define YL_CHECK(cond, st, ...)                         \
  do {                                                  \
    if (!(cond)) return ::yl::set_error(st, __VA_ARGS__); \
  } while (0)

#define YL_TRY(expr)               \
  do {                             \
    yl_status s_ = (expr);         \
    if (s_ != YL_OK) return s_;    \
  } while (0)

// Checks the launch that was just queued.
yl_status check_launch(const char* what);

inline unsigned grid_1d(size_t n, int block, int max_blocks = 148 * 32) {
  size_t g = (n + block - 1) / block;
  if (g < 1) g = 1;
  if (g > (size_t)max_blocks) g = max_blocks;
  return (unsigned)g;
}

}  // namespace yl

// The context: one device, one stream, a device error word, and a
// stream-ordered scratch buffer that ops carve their temporaries from.
struct yl_ctx {
  int device = 0;
  int num_sms = 148;
  cudaStream_t own_stream = nullptr;
  cudaStream_t stream = nullptr;
  cudaEvent_t ev_begin = nullptr;
  cudaEvent_t ev_end = nullptr;
  bool session_open = false;
  std::chrono::steady_clock::time_point wall_begin;
  // device control block (16 bytes): int error word at [0] (zeroed at
  // creation), long long bounded-wait limit in SM cycles at byte 8 (0 = the
  // kernels' default)
  int* dev_err = nullptr;
  // names of the last conv kernel templates launched on this context:
  // [0] forward / dX, [1] filter gradient (diagnostics, yl_ctx_last_kernel)
  char last_kernel[2][96] = {{0}, {0}};
  // FLOPs (2 x MACs) those launches executed, padding and merged taps as run
  double last_exec_flops[2] = {0.0, 0.0};
  // tile counters of the persistent conv kernels: kSchedSlots pairs (tiles
  // handed out, CTAs done), zero between launches; consecutive launches take
  // consecutive pairs so launches in flight together never share one
  int* sched = nullptr;
  unsigned sched_next = 0;
  // Scratch slots: 0 = temporaries of one internal kernel sequence (split-K
  // partials, reduction partials); 1 = layout conversions of a C-ABI call.
  // slot 0: operator temporaries; 1: NCHW<->NHWC staging of the batched
  // C-ABI entry points; 2: GroupNorm statistics partials written by a conv
  void* scratch[3] = {nullptr, nullptr, nullptr};
  size_t scratch_bytes[3] = {0, 0, 0};
  // workspace of the operators that take theirs through yl::Workspace, with an
  // event behind its last use
  void* work = nullptr;
  size_t work_bytes = 0;
  cudaEvent_t work_ev = nullptr;
  bool work_used = false;
  // largest cluster of the on-chip Newton-Schulz kernel; -1: not asked yet
  int chip_cluster = -1;
};

namespace yl {
constexpr int kSchedSlots = 64;

// Returns a device buffer of at least `bytes` from scratch slot `slot`,
// valid for work queued on ctx->stream until the next call on the same slot.
// Grows with cudaMallocAsync/cudaFreeAsync (stream-ordered, so a buffer
// still in use by queued work is never reused early).
yl_status scratch_get(yl_ctx* ctx, size_t bytes, void** out, int slot = 0);

// Makes the context's device current for one call and restores the caller's.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
    if (prev_ != device) {
      status_ = cudaSetDevice(device);
      restore_ = prev_ >= 0;
    }
  }
  ~DeviceGuard() {
    if (restore_) cudaSetDevice(prev_);
  }
  cudaError_t status() const { return status_; }

 private:
  int prev_ = -1;
  bool restore_ = false;
  cudaError_t status_ = cudaSuccess;
};

// Temporaries of one operator call.  Outside a stream capture they live in the
// context's workspace, and every call's work waits for that of the last one: by an
// event, whatever the stream handles, since a destroyed stream's handle may be given
// out again while its work still runs, and the per-thread default stream's is
// another stream in every host thread.  Inside a capture they are allocated and
// freed by nodes of the graph itself, so a graph neither keeps a pointer into the
// context's workspace (which may grow) nor shares it with another graph.
class Workspace {
 public:
  ~Workspace() { done(); }  // an early return must not leak a graph's allocation
  yl_status get(yl_ctx* ctx, size_t bytes, char** out);
  yl_status done();

 private:
  yl_ctx* ctx_ = nullptr;
  void* p_ = nullptr;
  bool captured_ = false;
};

// Bump allocator over one scratch buffer (256-byte aligned pieces).
struct ScratchCarver {
  size_t offset = 0;
  size_t take(size_t bytes) {
    size_t o = offset;
    offset += (bytes + 255) & ~size_t(255);
    return o;
  }
};
}  // namespace yl
