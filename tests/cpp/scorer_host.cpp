// The scorer's host code without a GPU: a shared library of the library's own
// objects over a device that only writes down what it is asked for and launchers
// that write down what they are given, for tests/test_scorer_host.py. Device
// addresses are numbers that nothing reads.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <string>

#include "jf_objects.h"
#include "jf_scorer.h"

namespace {
std::string g_log;  // one JSON object a line
int g_device = 0;
bool g_capturing = false;
uint64_t g_next = 1ull << 40;

void note(const char *what, const std::string &more = "") {
  g_log += "{\"what\": \"" + std::string(what) + "\"" + more + "}\n";
}
std::string number(const char *name, uint64_t v) {
  return ", \"" + std::string(name) + "\": " + std::to_string(v);
}
std::string address(const char *name, const void *p) { return number(name, (uint64_t)p); }
}  // namespace

extern "C" {

const char *fake_log() {
  static std::string taken;
  taken.swap(g_log);
  g_log.clear();
  return taken.c_str();
}
void fake_device(int device) { g_device = device; }
void fake_capturing(int capturing) { g_capturing = capturing != 0; }
// A penalty table of one row, on `device`.
jf_penalty_table *fake_penalty_table(uint32_t vocabulary, int device) {
  jf_penalty_table *t = new jf_penalty_table;
  t->vocabulary = vocabulary;
  t->rows = 1;
  t->max_entries = 1;
  t->device = device;
  t->stale.assign(1, 0);
  return t;
}
void fake_penalty_table_free(jf_penalty_table *t) { delete t; }

hipError_t hipGetDevice(int *device) {
  *device = g_device;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes) {
  *p = (void *)g_next;
  g_next += (bytes + 4095) / 4096 * 4096 + 4096;
  note("malloc", address("at", *p) + number("bytes", bytes));
  return hipSuccess;
}
hipError_t hipFree(void *p) {
  if (p) note("free", address("at", p));
  return hipSuccess;
}
hipError_t hipHostMalloc(void **p, size_t bytes, unsigned) {
  *p = std::malloc(bytes);
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipHostFree(void *p) {
  std::free(p);
  return hipSuccess;
}
hipError_t hipHostGetDevicePointer(void **device, void *host, unsigned) {
  *device = host;
  return hipSuccess;
}
hipError_t hipMemset(void *, int, size_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) {
  *e = (hipEvent_t)1;
  return hipSuccess;
}
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *to, const void *from, size_t bytes, hipMemcpyKind, hipStream_t) {
  std::string hex;
  for (size_t i = 0; i < bytes && i < 4096; ++i) {
    char digits[3];
    std::snprintf(digits, sizeof(digits), "%02x", ((const uint8_t *)from)[i]);
    hex += digits;
  }
  note("copy", address("to", to) + number("bytes", bytes) + ", \"held\": \"" + hex + "\"");
  return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *status) {
  *status = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "an error"; }

}  // extern "C"

namespace jf {

int launch_process(const ProcessLaunch &a, uint32_t, uint32_t, void *) {
  note("process", address("rows", a.rows) + number("row_count", a.row_count) +
                      number("any_masked", a.any_masked));
  return 0;
}

namespace {
int score_note(const char *what, const ScoreLaunch &a) {
  note(what, address("partials", a.partials) + address("aheads", a.aheads) +
                 address("maxima", a.maxima) + address("saved", a.saved) +
                 number("row_count", a.row_count) + number("segments", a.segments) +
                 number("groups", a.groups) + number("top", a.top));
  return 0;
}
}  // namespace
int launch_score(const ScoreLaunch &a, uint32_t, void *) { return score_note("score", a); }
int launch_logprobs(const ScoreLaunch &a, uint32_t, void *) { return score_note("logprobs", a); }
int launch_distill_loss(const ScoreLaunch &a, uint32_t, void *) { return score_note("loss", a); }
int launch_distill_grad(const DistillGradLaunch &a, uint32_t, void *) {
  note("grad", address("saved", a.saved) + number("row_count", a.row_count) +
                   number("teacher_count", a.teacher_count));
  return 0;
}
int launch_distill_step(const ScoreLaunch &a, const DistillGradLaunch &, uint32_t, void *) {
  return score_note("step", a);
}

}  // namespace jf
