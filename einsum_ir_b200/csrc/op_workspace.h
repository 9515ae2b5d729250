// Workspaces of the operators' plans (host only).
//
// The memory comes from a pool of the library's own per device, so that a plan made
// for a new shape does not pay for cudaMalloc on its first call (0.5 ms and more; it
// synchronises the device too). Up to 256 MiB stay with the pool when plans are
// destroyed.
#pragma once

#include <cuda_runtime_api.h>
#include <cstdint>
#include <mutex>
#include <new>
#include "eir_cuda.h"

namespace eir {

int api_set_error(int code, char const *msg);
int api_cuda_fail(cudaError_t e, char const *where);

inline int workspace_pool(int dev, cudaMemPool_t *pool) {
  static std::mutex mu;
  static cudaMemPool_t pools[64] = {};
  if (dev < 0 || dev >= 64) return api_set_error(EIR_CUDA_ERROR, "device index out of range");
  std::lock_guard<std::mutex> lk(mu);
  if (pools[dev] == nullptr) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = dev;
    cudaMemPool_t made = nullptr;
    cudaError_t e = cudaMemPoolCreate(&made, &props);
    if (e != cudaSuccess) return api_cuda_fail(e, "cudaMemPoolCreate");
    uint64_t keep = (uint64_t)256 << 20;
    e = cudaMemPoolSetAttribute(made, cudaMemPoolAttrReleaseThreshold, &keep);
    if (e != cudaSuccess) {
      cudaMemPoolDestroy(made);
      return api_cuda_fail(e, "cudaMemPoolSetAttribute");
    }
    pools[dev] = made;
  }
  *pool = pools[dev];
  return EIR_SUCCESS;
}

// A plan's own workspaces, one a device that it has been called on, each allocated on first use in
// `st`'s order and kept until release() (a graph captured on one device goes on using its memory
// there whatever the plan does on another). On another stream than the last use's a call waits for that. A
// capture gets the workspace that is there: memory allocated in it would be the graph's own, and an event from
// outside cannot be waited for (the caller orders a graph's launches).
class OpWorkspace {
 public:
  // A host thread holds the workspace from take(), before the launches that use the memory, to used(), behind
  // them: another one's call of the plan comes behind all of them
  std::unique_lock<std::mutex> hold() { return std::unique_lock<std::mutex>(mu_); }
  int take(int64_t bytes, cudaStream_t st, void **ws) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return api_cuda_fail(e, "cudaGetDevice");
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    e = cudaStreamIsCapturing(st, &cap);
    if (e != cudaSuccess) return api_cuda_fail(e, "cudaStreamIsCapturing");
    const bool captured = cap != cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (!captured) {
      e = cudaStreamGetId(st, &id);
      if (e != cudaSuccess) return api_cuda_fail(e, "cudaStreamGetId");
    }
    Memory *m = on(dev);
    if (m == nullptr) {
      if (captured)
        return api_set_error(EIR_INVALID_ARGUMENT,
                             "a plan with a workspace needs a call on the device before it is captured");
      int rc = allocate(bytes, dev, st, &m);
      if (rc != EIR_SUCCESS) return rc;
      m->stream = id;
    } else if (!captured && id != m->stream) {
      e = cudaStreamWaitEvent(st, m->used, 0);
      if (e != cudaSuccess) return api_cuda_fail(e, "cudaStreamWaitEvent(workspace)");
    }
    taken_ = m;
    id_ = id;
    captured_ = captured;
    *ws = m->ptr;
    return EIR_SUCCESS;
  }
  // marks the end of the use, which other streams and release() wait for; rc: the launches' status, returned
  int used(cudaStream_t st, int rc) {
    if (captured_) return rc;
    cudaError_t e = cudaEventRecord(taken_->used, st);
    if (e == cudaSuccess) taken_->stream = id_;
    return rc != EIR_SUCCESS || e == cudaSuccess ? rc : api_cuda_fail(e, "cudaEventRecord(workspace)");
  }
  void release() {
    int cur = 0;
    if (first_ != nullptr) cudaGetDevice(&cur);
    while (first_ != nullptr) {
      Memory *m = first_;
      first_ = m->next;
      if (m->device != cur) cudaSetDevice(m->device);
      cudaEventSynchronize(m->used);  // cudaFree of pool memory does not wait for its use
      cudaFree(m->ptr);
      cudaEventDestroy(m->used);
      if (m->device != cur) cudaSetDevice(cur);
      delete m;
    }
  }

 private:
  struct Memory {
    void *ptr = nullptr;
    int device = -1;
    cudaEvent_t used = nullptr;
    // of the last use: a stream's number, since handles are used again and the per-thread default stream has one
    // for all threads
    unsigned long long stream = 0;
    Memory *next = nullptr;
  };
  Memory *on(int dev) const {
    Memory *m = first_;
    while (m != nullptr && m->device != dev) m = m->next;
    return m;
  }
  int allocate(int64_t bytes, int dev, cudaStream_t st, Memory **made) {
    cudaMemPool_t pool = nullptr;
    int rc = workspace_pool(dev, &pool);
    if (rc != EIR_SUCCESS) return rc;
    Memory *m = new (std::nothrow) Memory;
    if (m == nullptr) return api_set_error(EIR_UNDEFINED_ERROR, "out of host memory");
    m->device = dev;
    char const *where = "cudaEventCreate(workspace)";
    cudaError_t e = cudaEventCreateWithFlags(&m->used, cudaEventDisableTiming);
    if (e == cudaSuccess) {
      where = "cudaMallocFromPoolAsync(workspace)";
      e = cudaMallocFromPoolAsync(&m->ptr, (size_t)bytes, pool, st);
      if (e != cudaSuccess) cudaEventDestroy(m->used);
    }
    if (e != cudaSuccess) {
      delete m;
      return api_cuda_fail(e, where);
    }
    m->next = first_;
    first_ = m;
    *made = m;
    // (another stream's call is ordered behind the allocation even if nothing uses the memory here)
    e = cudaEventRecord(m->used, st);
    return e == cudaSuccess ? EIR_SUCCESS : api_cuda_fail(e, "cudaEventRecord(workspace)");
  }

  std::mutex mu_;
  Memory *first_ = nullptr;
  // what the last take() found, for used()
  Memory *taken_ = nullptr;
  unsigned long long id_ = 0;
  bool captured_ = false;
};

}  // namespace eir
