"""The workspace and the error messages of operator calls (csrc/yl_runtime.cu) against
a stand-in for the CUDA runtime that writes down what is asked of it.

A stream handle does not name a stream for good: a destroyed stream's handle is
given out again while its work still runs, and the per-thread default stream's
handle is another stream in every thread.  So each use of the buffer, and its
release for a larger one, is ordered behind the last use whatever the handles."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "yumelayers_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>
#include <string>
#include <vector>
#include "yl_internal.h"

static std::vector<std::string> log_;
static bool capturing = false, no_memory = false;
static size_t next_buffer = 0x1000;
static void note(const char* what, const void* a, const void* b = nullptr) {
  char s[128];
  snprintf(s, sizeof s, "%s %lx %lx", what, (long)a, (long)b);
  log_.push_back(s);
}

extern "C" {
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
  *s = capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
cudaError_t cudaMallocAsync(void** p, size_t n, cudaStream_t s) {
  if (no_memory) return cudaErrorMemoryAllocation;
  *p = (void*)next_buffer;
  next_buffer += n;
  note("malloc", s);
  return cudaSuccess;
}
cudaError_t cudaFreeAsync(void*, cudaStream_t s) { note("free", s); return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = (cudaEvent_t)0xe; return cudaSuccess; }
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) { note("wait", s, e); return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { note("record", s, e); return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "stand-in"; }
}

static bool no_new = false;  // operator new fails
void* operator new(size_t n) {
  void* p = no_new ? nullptr : malloc(n);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

static void use(yl_ctx* ctx, size_t bytes) {
  yl::Workspace w;
  char* p = nullptr;
  const yl_status st = w.get(ctx, bytes, &p);
  if (st == YL_OK) note("use", ctx->stream);
  else note("status", (void*)(long)st);
  w.done();
}

int main(int, char** argv) {
  yl_ctx ctx;
  for (const char* c = argv[1]; *c; ++c) switch (*c) {
    case 'a': ctx.stream = (cudaStream_t)0xa; break;
    case 'b': ctx.stream = (cudaStream_t)0xb; break;
    case 's': use(&ctx, 1000); break;
    case 'l': use(&ctx, 100000); break;
    case 'c': capturing = !capturing; break;
    case 'm': no_memory = !no_memory; break;
    case 'e': {  // an error is reported where there is no host memory left
      no_new = true;
      const yl_status st = yl::set_error(YL_ERR_OOM, "no host memory for %d matrices, %2000d", 7, 8);
      const char* text = yl_last_error_message();
      no_new = false;
      printf("error %d %zu %.*s\n", (int)st, strlen(text), 24, text);
    }
  }
  for (const std::string& s : log_) puts(s.c_str());
}
"""

# what the rest of the file refers to, and this program never reaches
NEVER = ("cudaGetDeviceCount cudaSetDevice cudaGetDeviceProperties cudaStreamCreateWithFlags "
         "cudaEventCreate cudaMalloc cudaMemset cudaStreamSynchronize cudaEventSynchronize "
         "cudaEventDestroy cudaFree cudaStreamDestroy cudaEventQuery cudaEventElapsedTime "
         "cudaMemcpyAsync cudaMemsetAsync cudaGetDeviceProperties_v2").split()


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    d = tmp_path_factory.mktemp("workspace")
    (d / "program.cpp").write_text(PROGRAM)
    (d / "never.c").write_text("void abort(void);\n" + "".join(
        f"void {name}(void) {{ abort(); }}\n" for name in NEVER))
    subprocess.run(["gcc", "-c", str(d / "never.c"), "-o", str(d / "never.o")], check=True)
    subprocess.run(["g++", "-O0", "-std=c++17", "-I/usr/local/cuda/include", f"-I{CSRC}",
                    f"-I{ROOT / 'include'}", "-x", "c++", str(d / "program.cpp"),
                    str(CSRC / "yl_runtime.cu"), "-x", "none", str(d / "never.o"), "-o", str(d / "program")], check=True)

    def run(script):
        out = subprocess.run([d / "program", script], check=True, capture_output=True, text=True)
        return [line.split() for line in out.stdout.splitlines()]
    return run


@pytest.mark.parametrize("script", ["ass", "asl", "asbs", "asbl", "aslsl", "asbsas"])
def test_every_use_and_release_waits_for_the_last_use(calls, script):
    since_record, uses = None, 0
    for what, stream, event in calls(script):
        if what == "wait":
            assert event == "e"
            since_record = stream
        elif what in ("use", "free") and uses:
            assert since_record == stream, (what, stream)
        if what == "use":
            uses += 1
        if what == "record":
            since_record = None
    assert uses == sum(c in "sl" for c in script)


def test_captured_calls_take_and_free_their_own(calls):
    log = calls("ascscs")
    assert [w for w, *_ in log] == ["malloc", "use", "record", "malloc", "use", "free",
                                    "wait", "use", "record"]


def test_after_an_allocation_that_failed_the_next_call_takes_a_new_buffer(calls):
    log = [w for w, *_ in calls("asmlms")]
    assert log == ["malloc", "use", "record", "wait", "free", "status", "wait", "malloc", "use",
                   "record"]


def test_errors_are_reported_without_host_memory(calls):
    """A status that says there is no memory left takes none for its message."""
    (what, status, length, *text), = calls("e")
    assert what == "error" and int(length) == 1023
    assert " ".join(text) == "no host memory for 7 mat"
