"""yl_trainer_set_muon when host memory runs out: a program whose operator new fails
after a set number of calls asks again after every such failure, and its steps then
equal those of a trainer that had memory at once."""
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>
#include <vector>
#include "yume_c.h"

static long left = -1;  // allocations that still succeed; below 0: all
static void* take(size_t n) {
  if (left == 0) throw std::bad_alloc();
  if (left > 0) --left;
  void* p = malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void* operator new(size_t n) { return take(n); }
void* operator new[](size_t n) { return take(n); }
void operator delete(void* p) noexcept { free(p); }
void operator delete[](void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }
void operator delete[](void* p, size_t) noexcept { free(p); }

#define OK(expr)                                                                    \
  do {                                                                              \
    if ((expr) != YL_OK) {                                                          \
      printf("%s: %s\n", #expr, yl_last_error_message());                           \
      return 1;                                                                     \
    }                                                                               \
  } while (0)

static yl_ctx* ctx;
static const yl_muon_config kMuon = {0.02f, 0.02f, 0.95f, 1, 0.0f, 5};

static int stepped(yl_trainer* tr, std::vector<float>* out) {
  std::vector<float> frames(3 * 3 * 32 * 48), t(1, 0.5f);
  for (size_t i = 0; i < frames.size(); ++i) frames[i] = (float)(i * 7919 % 1000) / 1000.f;
  float losses[2];
  // two steps: the U-Net's last conv starts at zero, and what lies before it moves with
  // the second
  for (int k = 0; k < 2; ++k) OK(yl_trainer_step_host(tr, frames.data(), t.data(), losses));
  for (int which = 0; which < 2; ++which) {
    size_t n = 0;
    float* p = nullptr;
    OK(yl_trainer_param_count(tr, which, &n));
    OK(yl_trainer_buffer(tr, which, 0, &p));
    out[which].resize(n);
    OK(yl_memcpy_dtoh(ctx, out[which].data(), p, n * sizeof(float)));
  }
  return 0;
}

int main() {
  OK(yl_ctx_create(0, &ctx));
  yl_trainer_config cfg;
  memset(&cfg, 0, sizeof cfg);
  @CONFIG@
  std::vector<float> want[2], adam[2], got[2];
  yl_trainer* tr = nullptr;
  OK(yl_trainer_create(ctx, &cfg, nullptr, &tr));
  if (stepped(tr, adam)) return 1;
  OK(yl_trainer_destroy(tr));
  OK(yl_trainer_create(ctx, &cfg, nullptr, &tr));
  OK(yl_trainer_set_muon(tr, &kMuon));
  if (stepped(tr, want)) return 1;
  OK(yl_trainer_destroy(tr));
  OK(yl_trainer_create(ctx, &cfg, nullptr, &tr));
  int failures = 0;
  for (long n = 0;; ++n) {  // the n-th allocation of the call fails, then the call is made again
    left = n;
    const yl_status st = yl_trainer_set_muon(tr, &kMuon);
    const bool ran_out = left == 0;
    left = -1;
    if (st == YL_OK) break;
    if (st != YL_ERR_OOM || !ran_out) return printf("status %d after %ld\n", (int)st, n), 1;
    ++failures;
  }
  if (stepped(tr, got)) return 1;
  OK(yl_trainer_destroy(tr));
  OK(yl_ctx_destroy(ctx));
  for (int which = 0; which < 2; ++which) {
    if (got[which] != want[which]) return printf("model %d moved differently\n", which), 1;
    if (want[which] == adam[which]) return printf("model %d has no Muon\n", which), 1;
  }
  printf("failures %d\n", failures);
}
"""


def test_both_models_have_their_tables_after_memory_ran_out(tmp_path):
    from yumelayers_b200.trainer import default_config
    cfg = default_config(batch=1, height=32, width=48, seed=3)
    assigned = "\n".join(f"  cfg.{name} = {getattr(cfg, name)!r};" for name, _ in cfg._fields_)
    (tmp_path / "p.cpp").write_text(PROGRAM.replace("@CONFIG@", assigned))
    lib = ROOT / "yumelayers_b200"
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT / 'include'}", str(tmp_path / "p.cpp"), "-o",
                    str(tmp_path / "p"), f"-L{lib}", "-l:libyumecuda.so", f"-Wl,-rpath,{lib}"],
                   check=True)
    r = subprocess.run([tmp_path / "p"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    # a name's copy and several growths of either table's vectors
    assert int(r.stdout.split()[-1]) > 10
