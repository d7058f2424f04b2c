// lx_qwen2_set_prefill_bits where an allocation, a packing launch or the wait after it fails, against
// a stub of the HIP runtime on the host.  Prints "ok" or the first thing that is not as it should be.
// Built by tests/test_prefill_bits_alloc.py (host code only, no HIP runtime linked).
#include <cstdio>
#include <set>

#include "../../larynx_amd/csrc/lx_qwen2.cpp"

namespace {
std::set<void*> live;       // what hipMalloc gave and hipFree has not taken
int allocs_left = -1;       // -1: any number
int packs_left = -1;
bool sync_fails = false;
hipError_t last = hipSuccess;  // what hipGetLastError returns next
int freed_unknown = 0, device = 0, packed = 0;

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
hipError_t hipGetDevice(int* d) { return *d = device, hipSuccess; }
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
size_t lx_q8_bytes(int, int) { return 64; }
int lx_q8_pack_f32(const float*, long, const lx_q8*, hipStream_t) {
  if (packs_left == 0) {
    (void)hipGetLastError();  // as check_launch
    return LX_ERR_LAUNCH;
  }
  if (packs_left > 0) --packs_left;
  ++packed;
  return LX_OK;
}
}

namespace lx {
void set_error(const char*, ...) {}
}  // namespace lx

#define CHECK(what)                                    \
  do {                                                 \
    if (!(what)) {                                     \
      std::printf("%s (step %d)\n", #what, step);      \
      return 1;                                        \
    }                                                  \
  } while (0)

int main() {
  constexpr int kLayers = 3, kPacks = 1 + 4 * kLayers, kBuffers = kPacks + 2;
  int step = -1;
  lx_qwen2* m = new lx_qwen2();
  m->NL = kLayers;
  m->layers.resize(kLayers);
  m->device = 0;
  m->arena.alloc<float>(4);  // something of the model's own
  const auto own = live;
  auto as_it_was = [&]() {
    return live == own && m->arena.ptrs.size() == own.size() && last == hipSuccess &&
           !freed_unknown && !m->prefill8 && m->q8.layers.empty();
  };
  for (step = 0; step < kBuffers; ++step) {
    allocs_left = step;
    CHECK(lx_qwen2_set_prefill_bits(m, 8) == LX_ERR_ALLOC);
    CHECK(as_it_was());
    allocs_left = -1;
  }
  for (step = 0; step < kPacks; ++step) {
    packs_left = step;
    CHECK(lx_qwen2_set_prefill_bits(m, 8) == LX_ERR_LAUNCH);
    CHECK(as_it_was());
    packs_left = -1;
  }
  sync_fails = true;
  CHECK(lx_qwen2_set_prefill_bits(m, 8) == LX_ERR_LAUNCH);
  CHECK(as_it_was());
  sync_fails = false;
  device = 1;  // another device is current
  CHECK(lx_qwen2_set_prefill_bits(m, 8) == LX_ERR_ARG && as_it_was());
  device = 0;
  for (const int bits : {4, 0, 16, -8}) CHECK(lx_qwen2_set_prefill_bits(m, bits) == LX_ERR_ARG);
  CHECK(as_it_was());
  packed = 0;
  CHECK(lx_qwen2_set_prefill_bits(m, 8) == LX_OK && m->prefill8 && packed == kPacks);
  CHECK(live.size() == own.size() + kBuffers && (int)m->q8.layers.size() == kLayers);
  // packed once: the switch and back needs no memory
  allocs_left = packs_left = 0;
  for (const int bits : {32, 8, 8, 32, 8}) {
    CHECK(lx_qwen2_set_prefill_bits(m, bits) == LX_OK && m->prefill8 == (bits == 8));
    CHECK(live.size() == own.size() + kBuffers);
  }
  CHECK(lx_qwen2_set_prefill_bits(nullptr, 8) == LX_ERR_ARG);
  delete m;
  CHECK(live.empty() && !freed_unknown);
  std::puts("ok");
  return 0;
}
