// What the host sides of the C ABI's objects share: error returns, device
// allocations, the pinned buffers their uploads go through, and the penalty
// table, which both the selection and the processed logits read.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>
#include <string>
#include <vector>

#include "jf_host.h"
#include "jf_kernels.h"
#include "jf_sampler.h"

namespace jf::host {

inline int fail(int code, const std::string &message) { return jf::set_error(code, message); }

inline int hip_fail(hipError_t e, const char *what) {
  return fail(JF_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

#define JF_HIP(call, what)                       \
  do {                                           \
    const hipError_t e_ = (call);                \
    if (e_ != hipSuccess) return hip_fail(e_, what); \
  } while (0)

// Pinned host slots for asynchronous parameter uploads. A slot is reused
// only after the copy that last read it has completed.
class StagingRing {
 public:
  ~StagingRing() { release(); }

  int upload(void *device_dst, const void *src, size_t bytes,
             hipStream_t stream) {
    if (!bytes) return JF_OK;
    Slot &slot = slots_[next_];
    next_ = (next_ + 1) % kSlots;
    if (slot.pending) {
      JF_HIP(hipEventSynchronize(slot.event), "staging wait");
      slot.pending = false;
    }
    if (slot.capacity < bytes) {
      if (slot.host) JF_HIP(hipHostFree(slot.host), "staging free");
      slot.host = nullptr;
      slot.capacity = 0;
      size_t cap = 4096;
      while (cap < bytes) cap <<= 1;
      JF_HIP(hipHostMalloc(&slot.host, cap, hipHostMallocDefault),
             "staging alloc");
      slot.capacity = cap;
    }
    if (!slot.event)
      JF_HIP(hipEventCreateWithFlags(&slot.event, hipEventDisableTiming),
             "staging event");
    std::memcpy(slot.host, src, bytes);
    JF_HIP(hipMemcpyAsync(device_dst, slot.host, bytes, hipMemcpyHostToDevice,
                          stream),
           "parameter upload");
    JF_HIP(hipEventRecord(slot.event, stream), "staging record");
    slot.pending = true;
    return JF_OK;
  }

  void release() {
    for (Slot &slot : slots_) {
      if (slot.pending && slot.event) (void)hipEventSynchronize(slot.event);
      if (slot.event) (void)hipEventDestroy(slot.event);
      if (slot.host) (void)hipHostFree(slot.host);
      slot = Slot{};
    }
  }

 private:
  static constexpr int kSlots = 8;
  struct Slot {
    void *host = nullptr;
    size_t capacity = 0;
    hipEvent_t event = nullptr;
    bool pending = false;
  };
  Slot slots_[kSlots];
  int next_ = 0;
};

// Host-mapped buffers a kernel reads directly (coherent pinned memory, no
// copy): a slot is refilled only after the event recorded behind the last
// launch that read it has completed.
class MappedRing {
 public:
  ~MappedRing() { release(); }

  // A slot of at least `bytes` for the caller to fill at *host; *device
  // receives the address the kernel reads. Waits for the slot's last reader
  // and allocates before returning, so a failure leaves nothing changed.
  // record() must follow the launch.
  int acquire(size_t bytes, void **host, const void **device) {
    Slot &slot = slots_[next_];
    if (slot.pending) {
      JF_HIP(hipEventSynchronize(slot.event), "mapped batch wait");
      slot.pending = false;
    }
    if (slot.capacity < bytes) {
      if (slot.host) JF_HIP(hipHostFree(slot.host), "mapped batch free");
      slot.host = nullptr;
      slot.capacity = 0;
      size_t cap = 4096;
      while (cap < bytes) cap <<= 1;
      JF_HIP(hipHostMalloc(&slot.host, cap, hipHostMallocCoherent | hipHostMallocMapped),
             "mapped batch alloc");
      slot.capacity = cap;
      JF_HIP(hipHostGetDevicePointer(&slot.device, slot.host, 0), "mapped batch address");
    }
    if (!slot.event)
      JF_HIP(hipEventCreateWithFlags(&slot.event, hipEventDisableTiming), "mapped batch event");
    *host = slot.host;
    *device = slot.device;
    return JF_OK;
  }

  int record(hipStream_t stream) {
    Slot &slot = slots_[next_];
    next_ = (next_ + 1) % kSlots;
    JF_HIP(hipEventRecord(slot.event, stream), "mapped batch record");
    slot.pending = true;
    return JF_OK;
  }

  void release() {
    for (Slot &slot : slots_) {
      if (slot.pending && slot.event) (void)hipEventSynchronize(slot.event);
      if (slot.event) (void)hipEventDestroy(slot.event);
      if (slot.host) (void)hipHostFree(slot.host);
      slot = Slot{};
    }
  }

 private:
  static constexpr int kSlots = 4;
  struct Slot {
    void *host = nullptr;
    void *device = nullptr;
    size_t capacity = 0;
    hipEvent_t event = nullptr;
    bool pending = false;
  };
  Slot slots_[kSlots];
  int next_ = 0;
};

template <class T>
int device_alloc(T **p, size_t count, const char *what) {
  *p = nullptr;
  if (!count) return JF_OK;
  if (count > SIZE_MAX / sizeof(T))
    return fail(JF_ERR_NO_MEMORY, std::string(what) + ": more bytes than 64 bits count");
  JF_HIP(hipMalloc((void **)p, count * sizeof(T)), what);
  return JF_OK;
}

inline int check_device(int device) {
  int current = -1;
  JF_HIP(hipGetDevice(&current), "hipGetDevice");
  if (current != device)
    return fail(JF_ERR_INVALID_ARGUMENT,
                "call made on a different device than the object was created on");
  return JF_OK;
}

// Whether what is enqueued on `stream` goes into a graph now; the null stream's
// never does.
inline int is_capturing(hipStream_t stream, bool &capturing) {
  capturing = false;
  if (!stream) return JF_OK;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  JF_HIP(hipStreamIsCapturing(stream, &status), "capture status");
  capturing = status != hipStreamCaptureStatusNone;
  return JF_OK;
}

}  // namespace jf::host

// Fixed penalty slots a chunk at most (two per thread of the fast kernel).
constexpr uint32_t kMaxSlots = 2 * jf::kThreads;

struct jf_penalty_table {
  uint32_t vocabulary = 0;
  uint32_t rows = 0;
  uint32_t max_entries = 0;
  uint32_t buckets = 0;
  int device = 0;
  uint2 *entries = nullptr;    // [rows][max_entries] {token, word}
  uint32_t *offsets = nullptr; // [rows][buckets + 1]
  // The fast kernel's fixed slots: [rows][chunks][slot_count], 8192-token
  // chunks; host.fits(row) when every chunk of the row fits its slots and
  // every count fits the slot's 18 bits (otherwise select_kernel takes the
  // row). The array holds room for 512 slots a chunk; a table laid out 256
  // to a chunk widens to 512 when a row needs more (a history clustered in
  // one chunk's ids) and 512 suffice.
  uint32_t chunks = 0;
  uint32_t slot_count = 0;
  uint32_t *slots = nullptr;
  jf::PenaltyRows host;  // the rows as the device holds them
  // Rows a failed count may have left different on the device than in the
  // host copy: refused by jf_sample and by counts until rebuilt.
  std::vector<uint8_t> stale;
  jf::host::StagingRing staging;
  jf::host::MappedRing mapped;  // counts of more than kPenaltyOps tokens a call
};
