// Captured scratch of the operators between the linears (csrc/wq_scratch.cpp) on the CPU: the HIP calls it makes are the
// stand-ins below.  Prints one line per failed check; exit status 0 when there is none.
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <utility>
#include <vector>

#include "wq_scratch.h"

namespace {
constexpr size_t MB = (size_t)1 << 20;
int failed = 0, mallocs = 0;
size_t limit = (size_t)1 << 40, live = 0;
std::map<hipStream_t, unsigned long long> capturing;  // stream -> capture
unsigned long long captures = 0;
void expect(bool ok, const char* what) {
  if (!ok) printf("FAILED: %s\n", what), ++failed;
}
}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { return expect(capturing.empty(), "a synchronization in a capture"), hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
  expect(capturing.empty(), "an allocation in a capture");
  ++mallocs;
  if (live + n > limit) return hipErrorOutOfMemory;
  live += n;
  return (*p = calloc(1, n)) ? hipSuccess : hipErrorOutOfMemory;  // (untouched pages cost nothing)
}
hipError_t hipFree(void* p) { return free(p), hipSuccess; }
hipError_t hipMemset(void*, int, size_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* st) {
  return *st = capturing.count(s) ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipStreamGetCaptureInfo_v2(hipStream_t s, hipStreamCaptureStatus* st, unsigned long long* id, hipGraph_t*,
                                      const hipGraphNode_t**, size_t*) {
  if (hipStreamIsCapturing(s, st); *st == hipStreamCaptureStatusActive) *id = capturing[s];
  return hipSuccess;
}
}

using namespace agq;

namespace {
std::vector<std::pair<uint8_t*, uint8_t*>> taken;
bool apart(const CallScratch& c, size_t bytes) {
  uint8_t *const lo = reinterpret_cast<uint8_t*>(c.cnt), *const hi = c.data + bytes;
  bool ok = c.data >= lo + 4096;
  for (auto& t : taken) ok = ok && (hi <= t.first || t.second <= lo);
  taken.push_back({lo, hi});
  return ok;
}
hipStream_t stream(int i) { return reinterpret_cast<hipStream_t>((uintptr_t)0x1000 * (i + 1)); }
CallScratch captured(size_t bytes, ScratchOf of) {
  capturing[stream(2)] = ++captures;
  const CallScratch c = call_scratch(stream(2), bytes, of);
  capturing.clear();
  return c;
}
constexpr ScratchOf kLin = ScratchOf::kLinears, kOps = ScratchOf::kOperators;
}  // namespace

int main() {
  expect(!captured(MB, kOps).data && !captured(MB, kLin).data, "nothing before any other call");
  // a linear was called, no operator: these take from the first half of the linears' reserve
  call_scratch(stream(0), MB, kLin);
  int got = 0;
  for (int i = 0; i < 300; ++i)
    if (const CallScratch c = captured(MB, kOps); c.data) ++got, expect(apart(c, MB), "apart");
  expect(got > 100 && got <= 128, "operators leave the linears half");
  for (int i = 0; i < 100; ++i) {
    const CallScratch c = captured(MB, kLin);
    expect(c.data && apart(c, MB), "which they have");
  }
  // one graph a batch size, each called once before: all have scratch, twice over
  for (int twice = 0; twice < 2; ++twice)
    for (const size_t bytes : {16, 16, 16, 22, 43, 86, 172}) {
      expect(call_scratch(stream(1), bytes * MB, kOps).data, "a call");
      capturing[stream(2)] = ++captures;
      const CallScratch small = call_scratch(stream(2), 60 * MB, kOps), c = call_scratch(stream(2), bytes * MB, kOps);
      expect(small.data && c.data && apart(c, bytes * MB), "the captured call's own, beside a smaller one that came first");
      expect(bytes > 60 || small.data == c.data, "the calls of one capture share");
      const CallScratch lin = call_scratch(stream(2), 60 * 1024, kLin);
      expect(lin.data && apart(lin, 60 * 1024), "and beside the linears'");
      capturing.clear();
    }
  // what is there is enough: no further allocation
  const int before = mallocs;
  for (int i = 0; i < 20; ++i) call_scratch(stream(1), 100 * MB, kOps);
  expect(mallocs <= before + 1, "calls outside a capture allocate once");
  // the reserve ends
  got = 0;
  for (int i = 0; i < 60; ++i) {
    call_scratch(stream(1), 100 * MB, kOps);
    const CallScratch c = captured(100 * MB, kOps);
    if (c.data) ++got, expect(apart(c, 100 * MB), "apart to the end");
  }
  expect(got > 15 && got < 40, "4 GB in all");
  const int last = mallocs;
  call_scratch(stream(1), 100 * MB, kOps);
  expect(mallocs == last, "and no more");
  if (!failed) printf("scratch of the operators: all checks passed\n");
  return failed ? 1 : 0;
}
