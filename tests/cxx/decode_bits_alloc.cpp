// lx_qwen2_set_decode_bits where an allocation, a packing launch or the wait after it fails, against
// a stub of the HIP runtime on the host.  Prints "ok" or the first thing that is not as it should be.
// Built by tests/test_decode_bits_alloc.py (host code only, no HIP runtime linked).
#include <cstdio>
#include <set>

#include "../../larynx_amd/csrc/lx_qwen2.cpp"

namespace {
std::set<void*> live;       // what hipMalloc gave and hipFree has not taken
int allocs_left = -1;       // -1: any number
int packs_left = -1;
bool sync_fails = false;
hipError_t last = hipSuccess;  // what hipGetLastError returns next
int freed_unknown = 0;

hipError_t fail(hipError_t e) { return last = e; }
}  // namespace

extern "C" {
hipError_t hipMalloc(void** p, size_t) {
  if (allocs_left == 0) return fail(hipErrorOutOfMemory);
  if (allocs_left > 0) --allocs_left;
  live.insert(*p = new char);
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  if (!live.erase(p)) ++freed_unknown;
  else delete static_cast<char*>(p);
  return hipSuccess;
}
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) {
  return sync_fails ? fail(hipErrorLaunchFailure) : hipSuccess;
}
hipError_t hipGetLastError() {
  const hipError_t e = last;
  last = hipSuccess;
  return e;
}
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
}

namespace lx {
void set_error(const char*, ...) {}
size_t q4_bytes(int, int, int) { return 64; }
int q4_pack(const float*, void*, int, int, int, int, hipStream_t) {
  if (packs_left == 0) {
    (void)hipGetLastError();  // as check_launch
    return LX_ERR_LAUNCH;
  }
  if (packs_left > 0) --packs_left;
  return LX_OK;
}
}  // namespace lx

#define CHECK(what)                                    \
  do {                                                 \
    if (!(what)) {                                     \
      std::printf("%s (step %d)\n", #what, step);      \
      return 1;                                        \
    }                                                  \
  } while (0)

int main() {
  constexpr int kLayers = 3, kCopies = 1 + 3 * kLayers;
  int step = -1;
  lx_qwen2* m = new lx_qwen2();
  m->NL = kLayers;
  m->layers.resize(kLayers);
  m->device = 0;
  m->arena.alloc<float>(4);  // something of the model's own
  const auto own = live;
  auto as_it_was = [&](const std::set<void*>& mem) {
    return live == mem && m->arena.ptrs.size() == mem.size() && last == hipSuccess &&
           !freed_unknown;
  };
  for (step = 0; step < kCopies; ++step) {
    allocs_left = step;
    CHECK(lx_qwen2_set_decode_bits(m, 4, 64) == LX_ERR_ALLOC);
    CHECK(as_it_was(own) && !m->q4);
    allocs_left = -1;
    packs_left = step;
    CHECK(lx_qwen2_set_decode_bits(m, 4, 64) == LX_ERR_LAUNCH);
    CHECK(as_it_was(own) && !m->q4);
    packs_left = -1;
  }
  sync_fails = true;
  CHECK(lx_qwen2_set_decode_bits(m, 4, 64) == LX_ERR_LAUNCH);
  CHECK(as_it_was(own) && !m->q4);
  sync_fails = false;
  CHECK(lx_qwen2_set_decode_bits(m, 4, 64) == LX_OK);
  CHECK(live.size() == own.size() + kCopies && m->q4 && m->q4->group == 64);
  const auto with64 = live;
  // a group more that fails leaves the first in use, and its graphs
  m->graph[0] = reinterpret_cast<hipGraphExec_t>(m);
  for (step = 0; step < kCopies; ++step) {
    allocs_left = step;
    CHECK(lx_qwen2_set_decode_bits(m, 4, 32) == LX_ERR_ALLOC);
    CHECK(as_it_was(with64) && m->q4->group == 64 && m->graph[0]);
  }
  allocs_left = -1;
  for (const int group : {32, 128, 64, 32}) {
    CHECK(lx_qwen2_set_decode_bits(m, 4, group) == LX_OK && m->q4->group == group);
    CHECK(!m->graph[0] && m->q4->head && (int)m->q4->layers.size() == kLayers);
  }
  CHECK(live.size() == own.size() + 3 * kCopies);  // each group's set once
  CHECK(lx_qwen2_set_decode_bits(m, 32, 0) == LX_OK && !m->q4);
  delete m;
  CHECK(live.empty() && !freed_unknown);
  std::puts("ok");
  return 0;
}
